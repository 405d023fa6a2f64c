"""rotate_write on the GPU: rotated queries and keys, and keys and values in the cache, against the formula in 64 bits
and bit for bit against it in 32 (each product and sum rounded by itself); into 8- and 4-bit rows bit for bit."""
import pytest
import torch

import chunk_cases as C
import quant4_cases as Q
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

# lens, new, hq, hkv, d, bs, layers, dtype, rot, pairs
SHAPES = {
    "step": ([300, 1, 40], [1, 1, 1], 32, 8, 128, 16, 1, BF, 128, False),
    "round": ([300, 64, 33, 0], [120, 64, 0, 0], 8, 2, 128, 16, 3, BF, 128, False),
    "pairs": ([100, 20], [50, 7], 6, 2, 64, 32, 2, HF, 64, True),
    "part, halves": ([100, 20], [50, 7], 4, 2, 128, 16, 2, BF, 64, False),
    "part, pairs": ([100, 20], [50, 7], 4, 4, 64, 16, 2, HF, 32, True),
    "halves within a group": ([60], [60], 3, 1, 64, 16, 2, BF, 32, False),
    "fp32": ([100, 20], [50, 7], 3, 3, 96, 8, 1, FP, 96, False),
    "fp32 pairs": ([100, 20], [50, 7], 3, 1, 128, 8, 2, FP, 48, True),
    "head of 80": ([70, 90], [33, 1], 4, 2, 80, 16, 2, BF, 80, False),
    "odd sizes": ([37, 5], [20, 5], 3, 1, 50, 5, 2, BF, 22, False),
    "odd sizes, pairs": ([37, 5], [20, 5], 3, 1, 50, 5, 2, FP, 22, True),
    "wide head": ([40], [30], 2, 2, 256, 16, 1, BF, 256, False),
    "pairs of 128": ([100, 20], [50, 7], 4, 2, 128, 16, 2, BF, 128, True),
    "part, pairs of 128": ([100, 20], [50, 7], 4, 5, 128, 16, 2, BF, 80, True),
    "part of 80": ([100, 20], [50, 7], 7, 4, 80, 16, 3, BF, 40, False),
    "part of 80, pairs": ([100, 20], [50, 7], 7, 4, 80, 16, 3, HF, 40, True),
    "pieces of 4, fp32": ([70, 20], [50, 7], 3, 2, 72, 16, 2, FP, 24, False),
    "96, three heads": ([100, 20], [50, 7], 5, 3, 96, 16, 2, BF, 96, False),
    "96, pairs": ([100, 20], [50, 7], 5, 3, 96, 16, 2, HF, 48, True),
    "64, one head": ([100, 20], [50, 7], 1, 1, 64, 16, 4, HF, 64, False),
    "many tokens": ([2000, 700, 3], [1500, 700, 3], 8, 2, 128, 16, 2, BF, 128, False),
}


def _inputs(name, dev):
    from actkv_open_b200.kernels.rotary import rotary_table
    lens, new, hq, hkv, d, bs, layers, dtype, rot, pairs = SHAPES[name]
    table, nb, off, q, k, v, pos = Q.new_tokens(lens, new, hq, hkv, d, bs, layers, dtype, seed=len(name), positions=5000)
    angles = rotary_table(rot, 5000, device="cpu")
    return table, nb, off, q, k, v, pos, angles


def test_table_holds_the_angles():
    from actkv_open_b200.kernels.rotary import rotary_table
    t = rotary_table(64, 131072, base=500000.0, device="cpu").double()
    p = torch.tensor([0.0, 1.0, 77.0, 131071.0], dtype=torch.float64)
    f = 500000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    want = torch.cat([torch.cos(p[:, None] * f), torch.sin(p[:, None] * f)], 1)
    # one rounding to 32 bits of values up to 1
    assert (t[p.long()] - want).abs().max() <= 2.0 ** -24
    halved = rotary_table(64, 100, frequencies=f / 2, device="cpu").double()
    assert (halved[99] - torch.cat([torch.cos(99 * f / 2), torch.sin(99 * f / 2)])).abs().max() <= 2.0 ** -24


@pytest.mark.parametrize("name", SHAPES)
def test_cache_of_the_inputs_type(name):
    dev = need_gpu()
    from actkv_open_b200.kernels.rotary import rotate_write
    lens, new, hq, hkv, d, bs, layers, dtype, rot, pairs = SHAPES[name]
    table, nb, off, q, k, v, pos, angles = _inputs(name, dev)
    kv = torch.full((layers, 2, nb, bs, hkv, d), 7.0, dtype=dtype)
    got = kv.to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = rotate_write(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), angles.to(dev), off.to(dev), got, table.to(dev), seq,
                       interleaved=pairs)
    # in 32 bits, bit for bit
    assert torch.equal(out.cpu(), Q.turn(q.float(), pos, angles, pairs).to(dtype))
    turned = Q.turn(k.float(), pos, angles, pairs).to(dtype)
    tok, slot = Q.written(table, off, lens, bs, layers)
    flat = kv.view(layers, 2, nb * bs, hkv, d)
    flat[:, 0, slot], flat[:, 1, slot] = turned[:, tok], v[:, tok]
    assert torch.equal(got.cpu(), kv)
    # in 64 bits: two products, a sum (2^-24 of what they give each, at most 3 of |x| + |y|) and the last rounding
    for x, y in ((q, out.cpu()), (k, turned)):
        want = Q.turn(x.double(), pos, angles, pairs)
        room = 3 * 2.0 ** -24 * 2 * x.double().abs().amax(-1, keepdim=True) + torch.finfo(dtype).eps / 2 * want.abs() + \
            torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((y.double() - want).abs() <= room).all())
    assert_device_clean(dev)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("name", [n for n, s in SHAPES.items() if s[4] % 32 == 0])
def test_rows(name, bits):
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    from actkv_open_b200.kernels.rotary import rotate_write
    lens, new, hq, hkv, d, bs, layers, dtype, rot, pairs = SHAPES[name]
    table, nb, off, q, k, v, pos, angles = _inputs(name, dev)
    row = quant_row_bytes(hkv, d, bits)
    rows = torch.full((layers, 2, nb, bs, row), 0xAB, dtype=torch.uint8)
    got = rows.to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = rotate_write(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), angles.to(dev), off.to(dev), got, table.to(dev), seq,
                       interleaved=pairs, bits=bits)
    assert torch.equal(out.cpu(), Q.turn(q.float(), pos, angles, pairs).to(dtype))
    tok, slot = Q.written(table, off, lens, bs, layers)
    flat = rows.view(layers, 2, nb * bs, row)
    n = hkv * (d * bits // 8 + d // 32)
    pack = Q.pack_rows if bits == 4 else C.pack_rows
    for la in range(layers):
        for p, x in enumerate((Q.turn(k.float(), pos, angles, pairs), v)):
            flat[la, p, slot, :n] = pack(x[la, tok], row)[:, :n]
    assert torch.equal(got.cpu(), rows)
    assert_device_clean(dev)


def test_without_queries_in_place_and_other_strides():
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    from actkv_open_b200.kernels.rotary import rotate_write
    name = "part, halves"
    lens, new, hq, hkv, d, bs, layers, dtype, rot, pairs = SHAPES[name]
    table, nb, off, q, k, v, pos, angles = _inputs(name, dev)
    n = int(off[-1])
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    rest = (pos.to(dev), angles.to(dev), off.to(dev))
    kv = torch.zeros(layers, 2, nb, bs, hkv, d, dtype=dtype, device=dev)
    mine = q.to(dev)
    first = rotate_write(mine, k.to(dev), v.to(dev), *rest, kv, table.to(dev), seq)
    again = torch.zeros_like(kv)
    assert rotate_write(None, k.to(dev), v.to(dev), *rest, again, table.to(dev), seq) is None
    assert torch.equal(again, kv)
    assert rotate_write(mine, k.to(dev), v.to(dev), *rest, again, table.to(dev), seq, q_out=mine) is mine
    assert torch.equal(mine, first)
    # one tensor of q, k and v, off 16 bytes; angles with longer rows; caches of other strides
    both = torch.zeros(layers, n, (hq + 2 * hkv) * d + 1, dtype=dtype, device=dev)
    qkv = both[..., 1:].unflatten(-1, (hq + 2 * hkv, d))
    qkv.copy_(torch.cat([q, k, v], 2))
    wide = torch.zeros(5000, rot + 3, device=dev)[:, 1:rot + 1]
    wide.copy_(angles)
    cut = torch.zeros(layers, 2, nb, bs, hkv + 1, d + 1, dtype=dtype, device=dev)
    some = cut[..., 1:, 1:]
    out = torch.zeros(n, layers, hq, d + 1, dtype=dtype, device=dev)[..., :d].transpose(0, 1)
    rotate_write(qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:], rest[0], wide, rest[2], some, table.to(dev),
                 seq, q_out=out)
    assert torch.equal(out, first) and torch.equal(some, kv) and not cut[..., 0, :].any() and not cut[..., 0].any()
    for bits in (4, 8):
        row = quant_row_bytes(hkv, d, bits)
        a = torch.zeros(layers, 2, nb, bs, row, dtype=torch.uint8, device=dev)
        b = torch.zeros(layers, 2, nb, bs, row + 5, dtype=torch.uint8, device=dev)[..., 5:]
        rotate_write(None, k.to(dev), v.to(dev), *rest, a, table.to(dev), seq, bits=bits)
        rotate_write(qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:], rest[0], wide, rest[2], b, table.to(dev),
                     seq, bits=bits)
        assert torch.equal(a, b)
    assert_device_clean(dev)


@pytest.mark.parametrize("bits", [None, 8, 4])
@pytest.mark.parametrize("d", [128, 50])
def test_tokens_without_a_place_a_position_or_a_session(bits, d):
    dev = need_gpu()
    if bits and d % 32:
        pytest.skip("rows hold groups of 32")
    from actkv_open_b200 import _native as N
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    from actkv_open_b200.kernels.rotary import rotary_table, rotate_write
    lens, new, bs, hq, hkv = [40, 40, 20], [40, 8, 20], 16, 4, 2
    table, nb, off, q, k, v, pos = Q.new_tokens(lens, new, hq, hkv, d, bs, 1, BF, seed=3, positions=64)
    angles = rotary_table(d, 64)
    pad = 5                                              # rows behind the last session
    grow = lambda x: torch.cat([x, torch.ones(1, pad, *x.shape[2:], dtype=x.dtype)], 1).to(dev)  # noqa: E731
    pos = torch.cat([pos, torch.zeros(pad, dtype=torch.int32)])
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)

    def call(table, pos):
        if bits:
            cache = torch.full((1, 2, nb, bs, quant_row_bytes(hkv, d, bits)), 0xAB, dtype=torch.uint8, device=dev)
        else:
            cache = torch.full((1, 2, nb, bs, hkv, d), 7.0, dtype=BF, device=dev)
        out = torch.full((1, int(off[-1]) + pad, hq, d), 9.0, dtype=BF, device=dev)
        rotate_write(grow(q), grow(k), grow(v), pos.to(dev), angles, off.to(dev), cache, table.to(dev), seq, q_out=out, bits=bits)
        return out, cache.view(2, nb * bs, -1), N.read_device_status(dev)

    N.read_device_status(dev)
    out, cache, status = call(table, pos)
    assert status == 0 and bool((out[:, -pad:] == 9.0).all())
    bad_pos = pos.clone()
    bad_pos[3], bad_pos[45] = -1, 64
    o, c, status = call(table, bad_pos)
    assert status == N.DEV_BAD_INDEX and bool((o[:, [3, 45]] == 9.0).all())
    tok, slot = Q.written(table, off, lens, bs, 1)
    hit = (tok == 3) | (tok == 45)
    clean = torch.full_like(c[:, slot[hit]], 0xAB if bits else 7.0)
    assert torch.equal(c[:, slot[hit]], clean) and torch.equal(c[:, slot[~hit]], cache[:, slot[~hit]])
    rest = [i for i in range(out.shape[1]) if i not in (3, 45)]
    assert torch.equal(o[:, rest], out[:, rest])
    bad = table.clone()
    bad[0, 1], bad[2, 0] = -1, nb
    o, c, status = call(bad, pos)
    assert status == N.DEV_BAD_INDEX and torch.equal(o, out)
    hit = ((tok >= 16) & (tok < 32)) | ((tok >= 48) & (tok < 64))
    clean = torch.full_like(c[:, slot[hit]], 0xAB if bits else 7.0)
    assert torch.equal(c[:, slot[hit]], clean) and torch.equal(c[:, slot[~hit]], cache[:, slot[~hit]])


def test_nothing_new():
    dev = need_gpu()
    from actkv_open_b200.kernels.rotary import rotary_table, rotate_write
    e = torch.zeros(1, 0, 2, 64, dtype=BF, device=dev)
    kv = torch.zeros(1, 2, 2, 16, 2, 64, dtype=BF, device=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = rotate_write(e, e, e, i32(), rotary_table(64, 4), i32(0, 0), kv, i32(0).view(1, 1), i32(5))
    assert out.shape == e.shape and not kv.any()
    assert_device_clean(dev)
