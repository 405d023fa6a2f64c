"""The 4-bit cache on the GPU: rows written and read back bit for bit against the definition in 64 bits."""
import math

import pytest
import torch

import chunk_cases as C
import quant4_cases as Q
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

SHAPES = {
    "step": ([300, 1, 40], [1, 1, 1], 8, 128, 16, 3, BF),
    "round": ([300, 64, 33, 0], [120, 64, 0, 0], 8, 128, 16, 2, BF),
    "fp16": ([100, 20], [50, 7], 2, 64, 32, 2, HF),
    "fp32": ([100, 20], [50, 7], 3, 96, 8, 1, FP),
    "one narrow head": ([50], [50], 1, 32, 24, 2, BF),
    "wide head": ([50], [9], 2, 256, 16, 1, BF),
    "odd layers": ([70, 80], [9, 1], 4, 128, 16, 5, BF),
    "96": ([33, 80], [33, 1], 5, 96, 16, 2, BF),
    "96 fp16": ([33, 80], [33, 1], 8, 96, 16, 2, HF),
    "seven heads of 64": ([33, 80], [33, 1], 7, 64, 16, 1, FP),
}


def _empty(layers, nb, bs, hkv, d, row=None):
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    return torch.full((layers, 2, nb, bs, row or quant_row_bytes(hkv, d, 4)), 0xAB, dtype=torch.uint8)


def _want(rows, table, off, lens, bs, k, v):
    rows = rows.clone()
    layers, _, nb, _, row = rows.shape
    flat = rows.view(layers, 2, nb * bs, row)
    tok, slot = Q.written(table, off, lens, bs, layers)
    n = k.shape[2] * (k.shape[3] // 2 + k.shape[3] // 32)
    for la in range(layers):
        for p, x in enumerate((k, v)):
            flat[la, p, slot, :n] = Q.pack_rows(x[la, tok], row)[:, :n]
    return rows


@pytest.mark.parametrize("name", SHAPES)
def test_rows_written_and_read_back_bit_for_bit(name):
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    lens, new, hkv, d, bs, layers, dtype = SHAPES[name]
    table, nb, off, _, k, v, _ = Q.new_tokens(lens, new, hkv, hkv, d, bs, layers, dtype, seed=len(name))
    rows = _empty(layers, nb, bs, hkv, d)
    got, seq = rows.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    assert quantize_write(k.to(dev), v.to(dev), off.to(dev), got, table.to(dev), seq, bits=4) is got
    assert torch.equal(got.cpu(), _want(rows, table, off, lens, bs, k, v))
    args = (got, hkv, d, off.to(dev), table.to(dev), seq, int(off[-1]))
    rk, rv = dequantize_read(*args, dtype=dtype, bits=4)
    for x, y in ((rk, k), (rv, v)):
        assert torch.equal(x.cpu(), Q.quantise_ref(y)[0].to(dtype))
    only_k, none = dequantize_read(*args, dtype=dtype, planes="k", bits=4)
    assert none is None and torch.equal(only_k, rk)
    none, only_v = dequantize_read(*args, dtype=dtype, planes="v", bits=4)
    assert none is None and torch.equal(only_v, rv)
    assert_device_clean(dev)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_extreme_values(dtype):
    """Zeros of both signs, the type's largest and smallest, every level and every tie, scales at their edges, and
    groups with inf and NaN."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    sub = {BF: 2.0 ** -133, HF: 2.0 ** -24, FP: 2.0 ** -149}[dtype]
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.2, 5.1])
    groups = [torch.zeros(32), -torch.zeros(32), torch.cat([ties, -ties]), torch.cat([ties, -ties]) * 2.0 ** 9,
              torch.tensor([big] + [big / 3] * 31), torch.tensor([-big, tiny] * 16), torch.tensor([tiny, -sub] * 16),
              torch.tensor([sub, 3 * sub] * 16), torch.tensor([7.0] + [0.25] * 31), torch.tensor([7.03125] + [0.25] * 31),
              torch.tensor([math.inf] + [1.0] * 31), torch.tensor([1.0] * 31 + [math.nan]), torch.tensor([-math.inf, 0.0] * 16),
              torch.tensor([3.5 * 2.0 ** -5, 2.0 ** -14] * 16), torch.tensor([1e-3, 1e3] * 16), torch.tensor([6.0, -5.0] * 16)]
    x = torch.stack(groups).to(dtype).view(1, 4, 1, 128)
    off, lens = C.offsets([4]), [4]
    table = torch.zeros(1, 1, dtype=torch.int32)
    rows = _empty(1, 1, 16, 1, 128)
    got = rows.to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    quantize_write(x.to(dev), x.to(dev), off.to(dev), got, table.to(dev), seq, bits=4)
    assert torch.equal(got.cpu(), _want(rows, table, off, lens, 16, x, x))
    for out in (BF, HF, FP):
        k, v = dequantize_read(got, 1, 128, off.to(dev), table.to(dev), seq, 4, dtype=out, bits=4)
        want = Q.quantise_ref(x)[0]
        if out is HF:
            want = want.clamp(-65504.0, 65504.0)
        want = want.to(out)
        assert torch.equal(k.cpu().isnan(), want.isnan()) and torch.equal(k.cpu().nan_to_num(), want.nan_to_num())
        assert torch.equal(k.isnan(), v.isnan()) and torch.equal(k.nan_to_num(), v.nan_to_num())
    assert_device_clean(dev)


def test_any_scale_byte_reads_as_defined():
    """Rows that no writer made: every code under every scale byte, 253 and above NaN."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read
    rows = torch.zeros(1, 2, 16, 16, 32, dtype=torch.uint8)
    rows[..., :16] = (torch.arange(16) * 17).to(torch.uint8).flip(0)
    rows[..., 16] = torch.arange(256).view(16, 16).to(torch.uint8)
    table = torch.arange(16, dtype=torch.int32).view(1, 16).to(dev)
    off = torch.tensor([0, 256], dtype=torch.int32, device=dev)
    for out in (BF, HF, FP):
        k, _ = dequantize_read(rows.to(dev), 1, 32, off, table, off[1:], 256, dtype=out, bits=4)
        want = Q.unpack_rows(rows[0, 0].view(256, 32), 1, 32)
        if out is HF:
            want = want.clamp(-65504.0, 65504.0)
        want = want.to(out)
        assert torch.equal(k[0].cpu().isnan(), want.isnan()) and torch.equal(k[0].cpu().nan_to_num(), want.nan_to_num())
    assert_device_clean(dev)


def test_odd_strides_and_alignment():
    """Rows longer than they need be and off 16 bytes, inputs and outputs of other strides and off alignment."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    for d in (64, 96, 128):
        _odd(dev, d, dequantize_read, quantize_write)


def _odd(dev, d, dequantize_read, quantize_write):
    lens, new, hkv, bs = [40, 21], [33, 5], 3, 16
    table, nb, off, _, k, v, _ = Q.new_tokens(lens, new, 1, hkv, d, bs, 2, BF, seed=9)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    n = int(off[-1])
    least = hkv * (d // 2 + d // 32)
    for row, shift in ((least, 0), (least + 11, 3)):
        rows = _empty(2, nb, bs, hkv, d, row=row)
        flat = torch.full((rows.numel() + 8,), 0xCD, dtype=torch.uint8, device=dev)
        got = flat[shift:shift + rows.numel()].view(rows.shape)
        got.copy_(rows)
        kk = torch.zeros(2, hkv, n, d + 3, dtype=BF, device=dev)[..., 1:d + 1].transpose(1, 2)
        vv = torch.zeros(2, n + 2, hkv, d, dtype=BF, device=dev)[:, 2:]
        kk.copy_(k)
        vv.copy_(v)
        quantize_write(kk, vv, off.to(dev), got, table.to(dev), seq, bits=4)
        assert torch.equal(got.cpu(), _want(rows, table, off, lens, bs, k, v))
        assert bool((flat[:shift] == 0xCD).all()) and bool((flat[shift + rows.numel():] == 0xCD).all())
        out = torch.full((2, hkv, n, d + 3), 7.0, dtype=BF, device=dev)
        a, b = dequantize_read(got, hkv, d, off.to(dev), table.to(dev), seq, n, k_out=out[..., 1:d + 1].transpose(1, 2), bits=4)
        assert torch.equal(a.cpu(), Q.quantise_ref(k)[0].to(BF)) and torch.equal(b.cpu(), Q.quantise_ref(v)[0].to(BF))
        assert bool((out[..., 0] == 7.0).all()) and bool((out[..., d + 1:] == 7.0).all())
    assert_device_clean(dev)


def test_tokens_that_the_tables_do_not_hold_are_flagged_and_the_rest_written():
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    lens, new, bs = [40, 40, 20], [40, 8, 20], 16
    table, nb, off, _, k, v, _ = Q.new_tokens(lens, new, 1, 2, 64, bs, 1, BF, seed=3)
    bad = table.clone()
    bad[0, 1], bad[2, 0] = -1, nb
    rows = _empty(1, nb, bs, 2, 64)
    got = rows.to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    N.read_device_status(dev)
    pad = torch.zeros(1, 7, 2, 64, dtype=BF)             # rows behind the last session
    quantize_write(torch.cat([k, pad], 1).to(dev), torch.cat([v, pad], 1).to(dev), off.to(dev), got, bad.to(dev), seq, bits=4)
    assert N.read_device_status(dev) == N.DEV_BAD_INDEX
    want = _want(rows, table, off, lens, bs, k, v)
    want[0, :, table[0, 1].long()], want[0, :, table[2, 0].long()] = 0xAB, 0xAB
    assert torch.equal(got.cpu(), want)
    n = int(off[-1])
    out = torch.full((1, n + 7, 2, 64), 7.0, dtype=BF, device=dev)
    dequantize_read(got, 2, 64, off.to(dev), bad.to(dev), seq, n + 7, k_out=out, planes="k", bits=4)
    assert N.read_device_status(dev) == N.DEV_BAD_INDEX
    assert bool((out[:, 16:32] == 7.0).all()) and bool((out[:, 48:64] == 7.0).all()) and bool((out[:, n:] == 7.0).all())
    assert torch.equal(out[:, :16].cpu(), Q.quantise_ref(k[:, :16])[0].to(BF))
