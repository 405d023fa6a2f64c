"""PagedKVCache.chunk_attention checks its counts before anything reaches a GPU."""
import pytest
import torch

from actkv_open_b200.paged import PagedKVCache


@pytest.mark.parametrize("reqs, n_new, rows", [([0, 1], [2, 3], 4), ([0, 1], [2, 3], 6), ([0, 1], [5], 5), ([0], [2, 3], 5),
                                               ([0, 1], [6, -1], 5)])
def test_counts_that_are_not_the_queries_are_refused(reqs, n_new, rows):
    cache = PagedKVCache(8, 16, 2, 64)
    for r in (0, 1):
        cache.append(r, torch.zeros(1, 10, 2, 64), torch.zeros(1, 10, 2, 64))
    with pytest.raises(AssertionError, match="n_new"):
        cache.chunk_attention(reqs, torch.zeros(rows, 4, 64, dtype=torch.float16), n_new)
    with pytest.raises(RuntimeError, match="CUDA"):             # counts that fit go on to the kernels, which need a GPU
        cache.chunk_attention([0, 1], torch.zeros(5, 4, 64, dtype=torch.float16), [2, 3])
