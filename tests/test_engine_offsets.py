"""Offsets given as a tensor go to the kernels as they are: what is not on the cache's device, or not int32, is refused
before any launch (no GPU)."""
import pytest
import torch

from actkv_open_b200.engine import DevicePagedCache, QuantPagedCache


@pytest.mark.parametrize("kind", [DevicePagedCache, QuantPagedCache])
def test_host_offsets_are_refused(kind):
    cache = kind.__new__(kind)                   # (a cache of its own needs a GPU)
    cache.kv = torch.zeros(1, 2, 1, 16, 2, 64, dtype=torch.bfloat16)
    off = torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.reserve(off)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache._offsets(off)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_offsets_are_checked(bits):
    from gpu_util import assert_device_clean, need_gpu
    dev = need_gpu()
    c = DevicePagedCache(8, 16, 2, 64, 1, 2, 64, device=dev) if bits == 16 else \
        QuantPagedCache(8, 16, 2, 64, 1, 2, 64, device=dev, bits=bits)
    c.set_state([[], []], [0, 0], list(range(8)))
    k = torch.randn(1, 5, 2, 64, device=dev).bfloat16()
    good = torch.tensor([0, 2, 5], dtype=torch.int32, device=dev)
    for bad, error in ((good.cpu(), RuntimeError), (good.long(), AssertionError), (good[None], AssertionError),
                       (good[:0], AssertionError), (torch.stack([good, good], 1)[:, 0], AssertionError)):
        for call in (lambda x: c.reserve(x), lambda x: c.append(k, k, x, max_new=3)):
            with pytest.raises(error):
                call(bad)
    assert c.state()[1] == [0, 0]
    c.append(k, k, good, max_new=3)
    assert c.reserve(good) is good and c.state()[1] == [4, 6]
    assert_device_clean(dev)
