"""Argument checks of the rotation and of the 4-bit cache that need no GPU: status codes and messages before any
launch, refusals of the Python calls, and the layout arithmetic."""
import pytest
import torch

from actkv_open_b200 import _native as N
from actkv_open_b200.kernels.quant_cache import paged_chunk_attention_quant, quant_row_bytes, quantize_write
from actkv_open_b200.kernels.rotary import rotary_table, rotate_write


def _rotate(dtype=N.BF16, bits=0, rot=64, P=10, stride=64, Hq=4, Hkv=2, D=64, L=1, T=0, R=1, BS=16, row=4096, q=None):
    return N.load().actkv_rotate_write(q, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, dtype, None, None, stride, P,
                                       rot, 0, None, T, None, bits, 0, 0, 0, row, 0, None, 0, None, R, L, 1, 4, BS, Hq,
                                       Hkv, D, None, None)


def _write4(D=128, Hkv=2, row=4096, T=0):
    return N.load().actkv_quantize_write4(None, None, N.BF16, 0, 0, 0, 0, 0, 0, None, T, None, 0, 0, 0, row, None, 0, None,
                                          1, 1, 1, 4, 16, Hkv, D, None, None)


@pytest.mark.parametrize("call, match", [
    (lambda: _rotate(dtype=5), "dtype"), (lambda: _rotate(bits=16), "bits"), (lambda: _rotate(rot=0), "rotation"),
    (lambda: _rotate(rot=63), "rotation"), (lambda: _rotate(rot=66), "rotation"), (lambda: _rotate(P=0), "rotation"),
    (lambda: _rotate(stride=62), "shorter"), (lambda: _rotate(bits=4, rot=36), "multiples of 8"),
    (lambda: _rotate(bits=4, D=80), "multiple of 32"), (lambda: _rotate(bits=4, row=67), "shorter"),
    (lambda: _rotate(bits=8, row=131), "shorter"), (lambda: _rotate(T=3), "required"), (lambda: _rotate(Hq=-1), "sizes"),
    (lambda: _rotate(L=0), "sizes"), (lambda: _rotate(BS=0), "sizes"), (lambda: _rotate(L=1 << 22), "too many"),
    (lambda: _write4(D=48), "multiple"), (lambda: _write4(row=135), "shorter"), (lambda: _write4(T=2), "required"),
])
def test_bad_arguments_are_reported_before_any_launch(call, match):
    code = call()
    assert code == -1
    with pytest.raises(AssertionError, match=match):
        N.check(code)


def test_nothing_to_do_succeeds_without_a_device():
    assert _rotate() == 0 and _rotate(R=0, T=5) == 0 and _rotate(bits=4, row=68) == 0 and _write4(row=136) == 0


def test_row_sizes():
    assert quant_row_bytes(8, 128, 4) == 544 and quant_row_bytes(1, 64, 4) == 64 and quant_row_bytes(8, 64, 4) == 288
    assert quant_row_bytes(8, 128) == quant_row_bytes(8, 128, 8) == 1088
    with pytest.raises(ValueError, match="bits"):
        quant_row_bytes(8, 128, 2)
    with pytest.raises(AssertionError, match="multiple"):
        quant_row_bytes(8, 80, 4)


def test_python_refusals():
    k = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate_write(k, k, k, i32(0, 1, 2), rotary_table(64, 4, device="cpu"), i32(0, 3), torch.zeros(1, 2, 1, 16, 2, 64),
                     i32(0).view(1, 1), i32(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_write(k, k, i32(0, 3), torch.zeros(1, 2, 1, 16, 96, dtype=torch.uint8), i32(0).view(1, 1), i32(3), bits=4)
    with pytest.raises(ValueError, match="bits"):
        paged_chunk_attention_quant(k[0], i32(0, 3), torch.zeros(2, 1, 16, 96, dtype=torch.uint8), 2, i32(0).view(1, 1), i32(3),
                                    bits=16)
    for rot, positions in ((0, 4), (7, 4), (8, 0)):
        with pytest.raises(AssertionError):
            rotary_table(rot, positions, device="cpu")
    with pytest.raises(AssertionError, match="frequencies"):
        rotary_table(8, 4, frequencies=[1.0, 0.5], device="cpu")


def test_caches_hold_8_or_4_bits():
    from actkv_open_b200.engine import QuantPagedCache
    with pytest.raises(ValueError, match="bits 2"):
        QuantPagedCache(4, 16, 2, 128, 1, 1, 64, device="cpu", bits=2)
    with pytest.raises(ValueError, match="dtype"):
        QuantPagedCache(4, 16, 2, 128, 1, 1, 64, device="cpu", dtype=torch.float32, bits=4)
