"""The 8-bit cache on the GPU: rows written (quantize_write, actkv_quant_append) and read back
(dequantize_read), bit for bit against the definition in 64 bits, and QuantPagedCache through appends,
release and eviction."""
import math

import pytest
import torch

import chunk_cases as C
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _case(lens, new, hkv, d, bs, layers, dtype, seed, row=None):
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    gen = torch.Generator().manual_seed(seed)
    table, nb = C.pages(lens, bs, gen)
    off = C.offsets(new)
    n = int(off[-1])
    k = (torch.randn(layers, n, hkv, d, generator=gen) * torch.exp(3 * torch.randn(layers, n, hkv, 1, generator=gen))).to(dtype)
    v = torch.randn(layers, n, hkv, d, generator=gen).to(dtype)
    rows = torch.full((layers, 2, nb, bs, row or quant_row_bytes(hkv, d)), 0xAB, dtype=torch.uint8)
    return table, off, k, v, rows


def _want(table, off, k, v, rows, lens):
    rows = rows.clone()
    layers, _, nb, bs, row = rows.shape
    flat = rows.view(layers, 2, nb * bs, row)
    for r, s in enumerate(lens):
        o0, o1 = int(off[r]), int(off[r + 1])
        if o1 == o0:
            continue
        at = C.slots(table, r, s - (o1 - o0), s, bs)
        for la in range(layers):
            for p, x in enumerate((k, v)):
                packed = C.pack_rows(x[la, o0:o1], row)
                n = k.shape[2] * (k.shape[3] + k.shape[3] // 32)
                flat[la, p, at, :n] = packed[:, :n]
    return rows


SHAPES = {
    "step": ([300, 1, 40], [1, 1, 1], 8, 128, 16, 3, BF),
    "round": ([300, 64, 33, 0], [120, 64, 0, 0], 8, 128, 16, 2, BF),
    "fp16": ([100, 20], [50, 7], 2, 64, 32, 2, HF),
    "fp32": ([100, 20], [50, 7], 3, 96, 8, 1, FP),
    "one narrow head": ([50], [50], 1, 32, 24, 2, BF),
    "odd layers": ([70, 80], [9, 1], 4, 128, 16, 5, BF),
}


def _write(dev, case, lens):
    from actkv_open_b200.kernels.quant_cache import quantize_write
    table, off, k, v, rows = case
    got = rows.to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    quantize_write(k.to(dev), v.to(dev), off.to(dev), got, table.to(dev), seq)
    return got, seq


@pytest.mark.parametrize("name", SHAPES)
def test_rows_written_and_read_back_bit_for_bit(name):
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read
    lens, new, hkv, d, bs, layers, dtype = SHAPES[name]
    case = _case(lens, new, hkv, d, bs, layers, dtype, seed=len(name))
    table, off, k, v, _ = case
    got, seq = _write(dev, case, lens)
    assert torch.equal(got.cpu(), _want(*case, lens))
    rk, rv = dequantize_read(got, hkv, d, off.to(dev), table.to(dev), seq, int(off[-1]), dtype=dtype)
    for x, y in ((rk, k), (rv, v)):
        val, _, _ = C.quantise_ref(y)
        assert torch.equal(x.cpu(), val.to(dtype))
    only_k, none = dequantize_read(got, hkv, d, off.to(dev), table.to(dev), seq, int(off[-1]), dtype=dtype, planes="k")
    assert none is None and torch.equal(only_k, rk)
    none, only_v = dequantize_read(got, hkv, d, off.to(dev), table.to(dev), seq, int(off[-1]), dtype=dtype, planes="v")
    assert none is None and torch.equal(only_v, rv)
    assert_device_clean(dev)


def test_extreme_values():
    """Zeros, the type's largest and smallest, values at the scale's and the rounding's edges, and
    groups with inf and NaN, in bf16 and fp32."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read
    for dtype in (BF, FP):
        big = torch.finfo(dtype).max
        tiny = 2.0 ** -133 if dtype == BF else 2.0 ** -149
        groups = [[0.0], [big, -big, 1.0], [tiny, -tiny], [448.0, 1.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -11],
                  [450.0, 449.0], [448.0 * 2 ** -126, 2.0 ** -126], [448.0 * 2 ** -127], [math.inf, 1.0], [math.nan, 1.0],
                  [-math.inf], [17.0, 18.0, 19.0, 17.5, 18.5, -17.0, 240.0, 248.0, 232.0], [-0.0, 3.0]]
        x = torch.zeros(1, len(groups), 1, 32, dtype=torch.float64)
        for i, g in enumerate(groups):
            x[0, i, 0, :len(g)] = torch.tensor(g, dtype=torch.float64)
        x = x.to(dtype)
        n = len(groups)
        table, nb = C.pages([n], 16, torch.Generator().manual_seed(1))
        rows = torch.full((1, 2, nb, 16, 64), 0xAB, dtype=torch.uint8)
        case = (table, C.offsets([n]), x, x, rows)
        got, seq = _write(dev, case, [n])
        assert torch.equal(got.cpu(), _want(*case, [n]))
        rk, _ = dequantize_read(got, 1, 32, case[1].to(dev), table.to(dev), seq, n, dtype=FP)
        val, _, _ = C.quantise_ref(x)
        assert torch.equal(torch.nan_to_num(rk.cpu(), nan=77.0), torch.nan_to_num(val.float(), nan=77.0))
        assert torch.equal(torch.isnan(rk.cpu()), torch.isnan(val))
        # the error bound that the module states: 1/16 of the value, or half the smallest step
        fin = torch.isfinite(val)
        step = 2.0 ** -10 * torch.clamp(x.double().abs().amax(-1, keepdim=True) / 224, min=2.0 ** -127)
        assert ((val - x.double()).abs()[fin] <= torch.maximum(x.double().abs() / 16, step.expand_as(val))[fin]).all()
    assert_device_clean(dev)


def test_strided_rows_of_a_fused_projection_and_misaligned_caches():
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    lens, new = [60, 9], [33, 9]
    table, off, k, v, rows = case = _case(lens, new, 2, 64, 16, 2, BF, seed=5)
    want = _want(*case, lens)
    n = int(off[-1])
    fused = torch.zeros(n, 2, 3, 2, 64, dtype=BF, device=dev)            # token, layer, (q, k, v), head, dim
    fused[:, :, 1], fused[:, :, 2] = k.transpose(0, 1).to(dev), v.transpose(0, 1).to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    for shift in (0, 1, 4):                                              # bytes past a 16-byte boundary
        flat = torch.full((rows.numel() + 16,), 0xAB, dtype=torch.uint8, device=dev)
        got = flat[shift:shift + rows.numel()].view(rows.shape)
        quantize_write(fused[:, :, 1].transpose(0, 1), fused[:, :, 2].transpose(0, 1), off.to(dev), got, table.to(dev), seq)
        assert torch.equal(got.cpu(), want), shift
        wide = torch.zeros(2, n, 2, 65, dtype=BF, device=dev)            # rows that are not 16-byte aligned
        rk, rv = dequantize_read(got, 2, 64, off.to(dev), table.to(dev), seq, n, k_out=wide[..., 1:], v_out=None, dtype=BF)
        assert torch.equal(rk.cpu(), C.quantise_ref(k)[0].to(BF)) and torch.equal(rv.cpu(), C.quantise_ref(v)[0].to(BF))
        assert (wide[..., 0] == 0).all()
    assert_device_clean(dev)


def test_many_sessions():
    dev = need_gpu()
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 40, (100,), generator=g).tolist()
    new = [min(s, int(x)) for s, x in zip(lens, torch.randint(0, 9, (100,), generator=g))]
    case = _case(lens, new, 2, 64, 16, 2, BF, seed=6)
    got, _ = _write(dev, case, lens)
    assert torch.equal(got.cpu(), _want(*case, lens))
    assert_device_clean(dev)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: the last blocks of the last plane."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    lens, new = [40, 9], [40, 9]
    table, off, k, v, rows = case = _case(lens, new, 8, 128, 16, 1, BF, seed=7)
    first = (1 << 32) // (16 * rows.shape[-1]) + 1
    big = torch.zeros((1, 2, first + rows.shape[2]) + rows.shape[3:], dtype=torch.uint8, device=dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    t = (table + first).to(dev)
    big[:, :, first:] = 0xAB
    quantize_write(k.to(dev), v.to(dev), off.to(dev), big, t, seq)
    assert torch.equal(big[:, :, first:].cpu(), _want(*case, lens))
    assert not big[:, :, :first].any()
    rk, _ = dequantize_read(big, 8, 128, off.to(dev), t, seq, int(off[-1]))
    assert torch.equal(rk.cpu(), C.quantise_ref(k)[0].to(BF))
    assert_device_clean(dev)


def test_refusals():
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quant_row_bytes, quantize_write
    with pytest.raises(AssertionError):
        quant_row_bytes(2, 48)
    table, off, k, v, rows = (x.to(dev) for x in _case([20], [4], 2, 64, 16, 2, BF, seed=8))
    seq = torch.tensor([20], dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_write(k.cpu(), v, off, rows, table, seq)
    with pytest.raises(AssertionError):
        quantize_write(k, v.half(), off, rows, table, seq)
    with pytest.raises(AssertionError, match="layers"):
        quantize_write(k[:1], v[:1], off, rows, table, seq)
    with pytest.raises(AssertionError, match="short"):
        quantize_write(k, v, off, rows[..., :100], table, seq)
    with pytest.raises(AssertionError):
        quantize_write(k, v, off.long(), rows, table, seq)
    with pytest.raises(AssertionError):
        quantize_write(k[..., :48], v[..., :48], off, rows, table, seq)
    with pytest.raises(ValueError):
        dequantize_read(rows, 2, 64, off, table, seq, 4, planes="q")
    before = rows.clone()
    for t, s in ((torch.full_like(table, -1), seq), (torch.full_like(table, 1 << 30), seq),
                 (table, torch.tensor([3], dtype=torch.int32, device=dev)),
                 (table, torch.tensor([5000], dtype=torch.int32, device=dev))):
        one = before.clone()
        quantize_write(k, v, off, one, t, s)
        torch.cuda.synchronize()
        assert N.read_device_status(dev) == N.DEV_BAD_INDEX
        if s is seq:
            assert torch.equal(one, before)                               # nothing was written
    assert dequantize_read(rows, 2, 64, torch.zeros(2, dtype=torch.int32, device=dev), table, seq, 0)[0].shape[1] == 0
    assert_device_clean(dev)
