"""Argument checks of the chunk attention and 8-bit cache entry points that need no GPU: status codes
and messages before any launch, and the layout arithmetic."""
import pytest

from actkv_open_b200 import _native as N
from actkv_open_b200.kernels.quant_cache import quant_row_bytes


def _attend(dtype=N.BF16, T=0, R=1, MB=1, NB=4, BS=16, Hq=8, Hkv=2, D=128, scale=1.0, path=0, q=None, ws=None, wsb=0):
    return N.load().actkv_chunk_attention(q, dtype, 0, 0, None, T, None, 0, 0, 0, 0, None, 0, None, None, 0, 0, None, 0,
                                          R, MB, NB, BS, Hq, Hkv, D, scale, path, ws, wsb, None, None)


def _attend_quant(D=128, Hkv=2, row=4096, T=0):
    return N.load().actkv_chunk_attention_quant(None, N.BF16, 0, 0, None, T, None, 0, 0, row, None, 0, None, None, 0, 0,
                                                None, 0, 1, 1, 4, 16, 4 * Hkv, Hkv, D, 1.0, 0, None, 0, None, None)


def _write(dtype=N.BF16, D=128, Hkv=2, row=4096, T=0, L=1, BS=16):
    return N.load().actkv_quantize_write(None, None, dtype, 0, 0, 0, 0, 0, 0, None, T, None, 0, 0, 0, row, None, 0, None,
                                         1, L, 1, 4, BS, Hkv, D, None, None)


def _read(T=0, D=128):
    return N.load().actkv_dequantize_read(None, None, N.BF16, 0, 0, 0, 0, 0, 0, None, T, None, 0, 0, 0, 4096, None, 0,
                                          None, 1, 1, 1, 4, 16, 2, D, None, None)


@pytest.mark.parametrize("call, match", [
    (lambda: _attend(dtype=9), "dtype"), (lambda: _attend(Hq=7), "heads"), (lambda: _attend(Hkv=0), "heads"),
    (lambda: _attend(BS=0), "sizes"), (lambda: _attend(R=-1), "sizes"), (lambda: _attend(scale=0.0), "scale"),
    (lambda: _attend(path=3), "path"), (lambda: _attend(T=4), "required"),
    (lambda: _attend_quant(D=48), "multiple"), (lambda: _attend_quant(row=263), "shorter"),
    (lambda: _write(dtype=-1), "dtype"), (lambda: _write(D=40), "multiple"), (lambda: _write(row=263), "shorter"),
    (lambda: _write(L=0), "sizes"), (lambda: _write(BS=-1), "sizes"), (lambda: _write(T=3), "required"),
    (lambda: _read(D=33), "multiple"), (lambda: _read(T=3), "required"),
])
def test_bad_arguments_are_reported_before_any_launch(call, match):
    code = call()
    assert code == -1
    with pytest.raises(AssertionError, match=match):
        N.check(code)


def test_nothing_to_do_succeeds_without_a_device():
    assert _attend() == 0 and _attend(R=0) == 0 and _attend_quant() == 0 and _write() == 0 and _read() == 0


def test_workspace_and_row_sizes():
    assert N.load().actkv_chunk_workspace_bytes() % 256 == 0
    assert quant_row_bytes(8, 128) == 1088 and quant_row_bytes(1, 128) == 192 and quant_row_bytes(8, 64) == 576
    with pytest.raises(AssertionError):
        quant_row_bytes(8, 80)
