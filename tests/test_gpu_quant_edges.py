"""The 8-bit cache's writes and reads where offsets and types leave the ordinary."""
import pytest
import torch

import chunk_cases as C
from gpu_util import assert_device_clean, need_gpu
from test_gpu_quant_cache import BF, _case, _want, _write

pytestmark = pytest.mark.gpu


def test_rows_before_the_first_offset_are_no_sessions():
    """The last session of a batch by a slice of its offsets, k_new / v_new being the whole batch's: only that
    session's rows are written, and read back."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    lens, new = [60, 90], [33, 20]
    table, off, k, v, rows = case = _case(lens, new, 2, 64, 16, 2, BF, seed=9)
    whole = _want(*case, lens)
    at = C.slots(table, 1, 90 - 20, 90, 16)
    want = rows.clone()
    want.flatten(2, 3)[:, :, at] = whole.flatten(2, 3)[:, :, at]
    got = rows.to(dev)
    seq = torch.tensor(lens[1:], dtype=torch.int32, device=dev)
    quantize_write(k.to(dev), v.to(dev), off[1:].to(dev), got, table[1:].to(dev), seq)
    assert torch.equal(got.cpu(), want)
    full, seqs = _write(dev, case, lens)
    out = torch.full(k.shape, 3.0, dtype=BF, device=dev)
    dequantize_read(full, 2, 64, off[1:].to(dev), table[1:].to(dev), seqs[1:], 53, k_out=out, planes="k")
    assert (out[:, :33] == 3).all() and torch.equal(out[:, 33:].cpu(), C.quantise_ref(k)[0].to(BF)[:, 33:])
    assert_device_clean(dev)


def test_append_refuses_fewer_rows_than_new_tokens():
    """The counts are on the host: nothing is appended, where lengths would grow over rows that were never written."""
    dev = need_gpu()
    from actkv_open_b200.engine import QuantPagedCache
    c = QuantPagedCache(16, 16, 2, 64, 2, 2, 64, device=dev)
    c.set_state([[], []], [0, 0], list(range(16)))
    k = torch.ones(2, 20, 2, 64, dtype=BF, device=dev)
    c.append(k, k, [12, 8])
    state = c.state()
    with pytest.raises(AssertionError, match="rows"):
        c.append(k, k, [12, 9])
    assert c.state() == state
    c.append(k, k, [2, 3])                                # rows past the last count are no session's
    assert c.state()[1] == [14, 11]
    assert_device_clean(dev)
