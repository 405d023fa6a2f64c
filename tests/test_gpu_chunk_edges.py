"""Chunk attention where its schedule, its tables and its values leave the ordinary: units that see
nothing among units that do, both tensor-core kernels in one call, sessions of a few rows in every type
and head size, table entries and offsets out of range, values that are not finite.  Bounds as derived in
test_gpu_chunk.py."""
import pytest
import torch

import chunk_cases as C
from gpu_util import assert_device_clean, need_gpu
from test_gpu_chunk import BF, HF, Case, U, _equal

pytestmark = pytest.mark.gpu


def _empty_units(d, quant):
    """Sessions with many more new tokens than tokens (15 groups of 64 queries see nothing) between long
    ones: a CTA's share holds several units of both kinds, so a unit that leaves no product behind must not
    shift the waits of the units after it."""
    dev = need_gpu()
    lens, new = [10, 700, 0, 421] * 6, [1000, 150, 333, 131] * 6
    case = Case(lens, new, 8, 2, d, 16, BF, seed=21, quant=quant)
    x = case.device(dev)
    first = case.run(dev, given=x)
    case.check(first)
    for _ in range(3):
        assert _equal(first, case.run(dev, given=x))
    assert_device_clean(dev)


@pytest.mark.parametrize("d", [64, 128])
def test_units_that_see_nothing_among_units_that_do(d):
    _empty_units(d, quant=False)


@pytest.mark.parametrize("d", [64, 128])
def test_units_that_see_nothing_among_units_that_do_over_the_8_bit_cache(d):
    """Three and more such units in a row: the warp that brings scale bytes reads a tile ahead, and must
    not hold the last tile's while it looks for the next unit that has any."""
    _empty_units(d, quant=True)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("path", ["auto", "simt"])
@pytest.mark.parametrize("new, bad", [((2, 3, 2), (0, 2, 9, 9)), ((2, 90, 5), (0, 2, 92, 300)),
                                      ((4, 80, 5), (-3, 4, 84, 89)), ((2, 3, 2), (0, 2, 5, 1 << 30))])
def test_sessions_whose_offsets_leave_the_rows_are_left_alone(new, bad, path, quant):
    """Offsets past the last row of q, and below the first: flagged; the other sessions have their results, and
    nothing is written for the one that is out of range, inside the call's rows or past them."""
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    case = Case([500, 300, 40], list(new), 8, 2, 128, 16, BF, seed=22, quant=quant)
    t = sum(new)
    want = case.run(dev, path=path)
    room = torch.full((t + 400, 8, 128), 3.0, dtype=BF, device=dev), torch.full((t + 400, 8), 3.0, device=dev)
    off = torch.tensor(bad, dtype=torch.int32, device=dev)
    case.run(dev, given=dict(q_off=off), path=path, out=room[0][200:200 + t], lse=room[1][200:200 + t])
    torch.cuda.synchronize()
    assert N.read_device_status(dev) == N.DEV_BAD_INDEX
    written = torch.zeros(t + 400, dtype=torch.bool, device=dev)
    for a, b in zip(bad, bad[1:]):
        if 0 <= a < b <= t:
            rows = slice(200 + a, 200 + b)
            written[rows] = True
            if (a, b) in list(zip(case.off.tolist(), case.off.tolist()[1:])):
                assert all((x[rows] - y[a:b]).abs().max() <= 0.02 for x, y in zip(room, want))
    assert (room[0][~written] == 3).all() and (room[1][~written] == 3).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("path", ["auto", "simt"])
def test_rows_before_the_first_offset_are_no_sessions(path, quant):
    """The last sessions of a batch by a slice of its offsets, q being the whole batch's: the rows of the sessions
    that were left out are not written."""
    dev = need_gpu()
    case = Case([500, 300, 40], [6, 70, 3], 8, 2, 128, 16, BF, seed=23, quant=quant)
    x = case.device(dev)
    want = case.run(dev, given=x, path=path)
    out, lse = torch.full_like(want[0], 3.0), torch.full_like(want[1], 3.0)
    case.run(dev, given=dict(q_off=x["q_off"][2:], table=x["table"][2:], seq=x["seq"][2:]), path=path, out=out, lse=lse)
    assert (out[:76] == 3).all() and (lse[:76] == 3).all()
    # the same session may run on another kernel in the smaller batch: equal within twice the bound of one
    assert ((out[76:].double() - want[0][76:].double()).abs() <= 2 * (2 * U[BF] + 1e-4) * case.ref()[2].to(dev)[76:]).all()
    assert (lse[76:] - want[1][76:]).abs().max() <= 1e-3
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("bad", [-2, -3, -(1 << 31), (1 << 31) - 1])
def test_every_block_id_outside_the_cache_is_flagged(bad, new, quant):
    """One bad entry in the middle of a session's table, on the kernel for few rows, the wide one and the CUDA cores."""
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    case = Case([500], [new], 8, 4, 128, 16, BF, seed=24, quant=quant)
    x = case.device(dev)
    x["table"][0, 7] = bad
    for path in ("auto", "simt"):
        case.run(dev, given=x, path=path)
        torch.cuda.synchronize()
        assert N.read_device_status(dev) == N.DEV_BAD_INDEX


def _holes_ref(case, gone):
    """64-bit attention of a one- or many-session case in which the tokens gone[r] (a bool per token) are hidden."""
    t, hq, d = case.q.shape
    out, mag = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, d, dtype=torch.float64)
    lse, size = torch.full((t, hq), -torch.inf, dtype=torch.float64), torch.zeros(t, hq, dtype=torch.float64)
    for r, s in enumerate(case.lens):
        o0, o1 = int(case.off[r]), int(case.off[r + 1])
        k, v = (case.tokens(p, r).double().repeat_interleave(hq // case.hkv, 1) for p in range(2))
        q = case.q[o0:o1].double()
        x = torch.einsum("ahd,shd->ahs", q, k) * d ** -0.5
        hide = (torch.arange(s)[None] > torch.arange(s - (o1 - o0), s)[:, None]) | gone[r][None]
        x = x.masked_fill(hide[:, None], -torch.inf)
        one = torch.logsumexp(x, -1)
        p = torch.where(torch.isfinite(one)[..., None], torch.exp(x - one[..., None]), torch.zeros_like(x))
        out[o0:o1], mag[o0:o1] = (torch.einsum("ahs,shd->ahd", p, y) for y in (v, v.abs()))
        lse[o0:o1], size[o0:o1] = one, torch.einsum("ahd,shd->ahs", q.abs(), k.abs()).amax(-1) * d ** -0.5
    return out, lse, mag, size


def _within(got, ref):
    out, lse = (x.cpu().double() for x in got)
    want, want_l, mag, size = ref
    assert ((out - want).abs() <= (2 * U[BF] + 1e-4) * mag).all()
    empty = want_l == -torch.inf
    assert torch.equal(lse == -torch.inf, empty) and (out[empty] == 0).all()
    assert ((lse - want_l).abs()[~empty] <= 2e-5 + 8e-6 * size[~empty]).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("lens, new, bs, d", [([500], [1], 16, 128), ([500], [3], 16, 64), ([500, 300], [90, 2], 16, 128),
                                              ([700, 129], [300, 33], 64, 64), ([9000], [2], 16, 128),
                                              ([9000, 60], [70, 4], 16, 128), ([900], [140], 256, 128)])
def test_tokens_of_blocks_outside_the_cache_are_hidden(lens, new, bs, d, quant):
    """A bad entry at a table's start, middle and end, a whole bad row, and a table narrower than its session, on the
    tensor cores and the CUDA cores: those tokens count for nothing, and what block 0 holds (NaN here) is not read in
    their place."""
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    case = Case(lens, new, 8, 4, d, bs, BF, seed=25, quant=quant)
    x = case.device(dev)
    nan = 255 if quant else float("nan")
    x["cache"] = torch.cat([torch.full_like(x["cache"][:, :1], nan), x["cache"]], 1)
    whole = x["table"] + 1
    n = [-(-s // bs) for s in lens]
    for bad in ([0], [n[0] // 2], [n[0] - 1], [0, n[0] // 3, n[0] - 2], list(range(n[0])), "narrow"):
        gone = [torch.zeros(s, dtype=torch.bool) for s in lens]
        if bad == "narrow":
            keep = n[0] - 1 - n[0] // 4
            table = whole[:, :keep]
            for g in gone:
                g[keep * bs:] = True
            if keep == 0:
                continue
        else:
            table = whole.clone()
            for b in bad:
                table[0, b] = -1 if b % 2 else case.nb + 1 + b
                gone[0][b * bs:(b + 1) * bs] = True
        ref = _holes_ref(case, gone)
        for path in ("auto", "simt"):
            _within(case.run(dev, given={**x, "table": table}, path=path), ref)
            torch.cuda.synchronize()
            assert N.read_device_status(dev) == N.DEV_BAD_INDEX


def _one_token_sessions(byte, scale, plane, hkv, d, dtype, new):
    """R sessions of one token; its row of ``plane`` (0: keys, 1: values) has the given e4m3 bytes [R, Hkv, D] and scale
    bytes [R, Hkv, D / 32], the other plane's row is zero.  ``new`` query tokens each, the last of which sees the token;
    q is one-hot, of 1.  Returns the case and the dim [R * new, Hq] in which q is 1."""
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    r = byte.shape[0]
    case = Case.__new__(Case)
    case.lens, case.new, case.hq, case.hkv, case.d, case.bs, case.dtype, case.quant = [1] * r, [new] * r, 2 * hkv, hkv, d, 16, dtype, True
    case.table, case.nb = torch.arange(r, dtype=torch.int32)[:, None], r
    case.off = torch.arange(r + 1, dtype=torch.int32) * new
    case.row = quant_row_bytes(hkv, d)
    case.cache = torch.full((2, r, 16, case.row), 255, dtype=torch.uint8)
    case.cache[:, :, 0] = 0
    case.cache[plane, :, 0, :hkv * d] = byte.reshape(r, -1)
    case.cache[plane, :, 0, hkv * d:hkv * (d + d // 32)] = scale.reshape(r, -1)
    hot = (torch.arange(r * new)[:, None] * 7 + torch.arange(2 * hkv)[None] * 3) % d
    case.q = torch.nn.functional.one_hot(hot, d).to(dtype)
    return case, hot


def _read_back(case, dev):
    from actkv_open_b200.kernels.quant_cache import dequantize_read
    x = case.device(dev)
    r = len(case.lens)
    off = torch.arange(r + 1, dtype=torch.int32, device=dev)
    k, v = dequantize_read(x["cache"][None], case.hkv, case.d, off, x["table"], x["seq"], r, dtype=case.dtype)
    return k[0], v[0]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new, path", [(1, "auto"), (20, "auto"), (1, "simt")])
def test_every_scale_byte_is_attended_as_it_is_read_back(new, path, d, dtype):
    """One token per session: with a zero key the output is its value row bit for bit, and with one-hot queries the lse
    is a dim of its key, which shows what the attention kernels make of e4m3 bytes and scale bytes.  Scale bytes
    0 to 254 for the values (fp16: results that round to subnormals, to zero and past the range, which
    saturate; bf16 short of inf), and for keys those of logits up to 2^24."""
    dev = need_gpu()
    hkv, r = 2, 256
    gen = torch.Generator().manual_seed(26)
    byte = torch.randint(0, 256, (r, hkv, d), generator=gen)
    byte = torch.where((byte & 127) == 127, byte - 1, byte).to(torch.uint8)      # e4m3's own NaN is not of this test
    scale = torch.randint(0, 255, (r, hkv, d // 32), generator=gen)
    scale[:255, 0, 0] = torch.arange(255)
    scale[:60, 1, 0] = torch.arange(90, 150)
    last = torch.arange(r, device=dev) * new + new - 1
    most = (245, 142) if dtype == BF else (254, 254)
    case, _ = _one_token_sessions(byte, scale.clamp(max=most[0]), 1, hkv, d, dtype, new)
    out, lse = case.run(dev, path=path)
    assert torch.equal(out[last], _read_back(case, dev)[1].repeat_interleave(2, 1)) and (lse[last] == 0).all()
    case, hot = _one_token_sessions(byte, scale.clamp(max=most[1]), 0, hkv, d, dtype, new)
    out, lse = case.run(dev, path=path, scale=1.0)
    want = _read_back(case, dev)[0].repeat_interleave(2, 1).gather(2, hot.to(dev)[last][..., None])[..., 0].double()
    assert ((lse[last].double() - want).abs() <= 1e-6 * want.abs()).all() and (out[last] == 0).all()
    assert_device_clean(dev)


@pytest.mark.parametrize("new, path", [(3, "auto"), (90, "auto"), (200, "auto"), (3, "simt"), (90, "simt")])
@pytest.mark.parametrize("lens", [500, 5000])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_values_past_the_range_of_an_8_bit_cache(d, lens, new, path):
    """A value e4m3 * 2^(byte - 127) past bf16's range is inf, of either sign: rows that see its token have it in that
    dim, rows that do not (their p is 0) are as without it."""
    dev = need_gpu()
    case = Case([lens], [new], 8, 4, d, 16, BF, seed=27, quant=True)
    clean = case.run(dev, path=path)
    tok = lens - new + new // 2                          # the second half of the new tokens sees it
    at = int(C.slots(case.table, 0, tok, tok + 1, 16))
    head, dim = 2, 37
    group = slice(4 * d + (head * d + 32) // 32, 4 * d + (head * d + 32) // 32 + 1)
    lo = head * d + 32
    case.cache[1, at, lo:lo + 32] = 0
    case.cache[1, at, group] = 127
    zero = case.run(dev, path=path)                      # the same without those 32 values
    case.cache[1, at, head * d + dim], case.cache[1, at, head * d + dim + 1] = 0x7e, 0xfe
    case.cache[1, at, group] = 254
    got = case.run(dev, path=path)
    see, q = new // 2, slice(2 * head, 2 * head + 2)
    assert _equal([x[:see] for x in got], [x[:see] for x in clean]) and torch.equal(got[1], clean[1])
    assert (got[0][see:, q, dim] == torch.inf).all() and (got[0][see:, q, dim + 1] == -torch.inf).all()
    want = zero[0].clone()
    want[see:, q, dim], want[see:, q, dim + 1] = torch.inf, -torch.inf
    assert torch.equal(got[0], want)
    assert_device_clean(dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new, path", [(1, "auto"), (3, "auto"), (90, "auto"), (200, "auto"), (3, "simt")])
@pytest.mark.parametrize("lens", [500, 6000])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_among_e4m3_bytes_is_attended_as_it_is_read_back(d, lens, new, path, dtype):
    """Bytes 0x7f and 0xff read back as NaN: a value makes its dim of every row that sees it NaN, a key every dim
    and the lse, of its head's queries and of no others, wherever the token lies: among the first tokens, in the
    middle (all rows see it) and among the new ones (some do)."""
    dev = need_gpu()
    case = Case([lens, 40], [new, 1], 8, 4, d, 16, dtype, seed=28, quant=True)
    clean = case.run(dev, path=path)
    head, dim = 2, 37
    q, others = slice(2 * head, 2 * head + 2), [0, 1, 2, 3, 6, 7]
    rows = case.cache.clone()
    for tok in sorted({0, lens // 2 + 3, lens - new + new // 2}):
        at = int(C.slots(case.table, 0, tok, tok + 1, 16))
        see = max(0, tok - (lens - new))
        for plane, byte in ((1, 0x7f), (1, 0xff), (0, 0x7f), (0, 0xff)):
            case.cache = rows.clone()
            case.cache[plane, at, head * d + dim] = byte
            out, lse = case.run(dev, path=path)
            assert torch.equal(out[:, others], clean[0][:, others]) and torch.equal(lse[:, others], clean[1][:, others])
            assert _equal((out[:see], lse[:see]), [x[:see] for x in clean]) and _equal((out[new:], lse[new:]), [x[new:] for x in clean])
            if plane == 0:
                assert torch.isnan(out[see:new, q]).all() and torch.isnan(lse[see:new, q]).all()
            else:
                assert torch.isnan(out[see:new, q, dim]).all() and torch.equal(lse, clean[1])
                rest = [x for x in range(d) if x != dim]
                assert torch.equal(out[:, q][..., rest], clean[0][:, q][..., rest])
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("new", [1, 3, 90, 200])
def test_fp16_keeps_what_a_dominant_token_leaves(new, quant):
    """One token 17.4 above all others (an attention sink), with a zero value: the output is what 2000 others of
    p = e^-17.4 = 2^-25.1 add up to, half of fp16's smallest number each.  p is held in fp16 times 2^7 at least, so it
    errs by u of itself or 2^-25 / 2^7 = 2^-32 absolutely: |out - ref| <= (2 u + 1e-4) A + S 2^-32 max|v|, and the output's own
    subnormals err by 2^-25."""
    dev = need_gpu()
    s = 2000
    case = Case([s], [new], 4, 2, 128, 16, HF, seed=29, quant=quant)
    case.q.zero_()
    case.q[..., 0] = 17.4 / 18
    k, v = torch.zeros(s, 2, 128, dtype=HF), torch.ones(s, 2, 128, dtype=HF)
    k[0, :, 0], v[0] = 18, 0                             # 18 is exact in e4m3 too
    at = C.slots(case.table, 0, 0, s, 16)
    for p, x in enumerate((k, v)):
        case.cache[p, at] = C.pack_rows(x, case.row) if quant else x
    out, lse = (x.cpu().double() for x in case.run(dev, scale=1.0))
    want, want_l, mag, size = case.ref(1.0)
    assert (want < 1e-4).all() and (want > 2e-5).all()
    assert ((out - want).abs() <= (2 * U[HF] + 1e-4) * mag + s * 2.0 ** -32 + 2.0 ** -25).all()
    assert ((lse - want_l).abs() <= 2e-5 + 8e-6 * size).all()
    assert_device_clean(dev)


# ---------------------------------------------------------------- the kernel for few rows, and both kernels in one call

FEW = {   # lens, new, hq, hkv, block size: at most 16 rows (token x head of the group) per KV head; 8 over the 8-bit cache
    "one row": ([700, 129, 128, 127, 1, 2000, 40], [1] * 7, 8, 8, 16),
    "four of two": ([700, 129, 128, 127, 1, 2000, 0], [4, 1, 3, 2, 4, 4, 1], 8, 4, 16),
    "two of four": ([700, 17, 16, 15, 3000, 2], [2, 1, 2, 0, 2, 2], 32, 8, 32),
    "two of three": ([333, 64, 1000], [2, 1, 2], 6, 2, 8),
    "eight of one": ([500, 8, 3, 1200], [8, 8, 8, 5], 3, 3, 64),
    "one of five, one KV head": ([900, 33], [1, 1], 5, 1, 16),
    "one of eight": ([900, 33, 2500], [1, 1, 1], 32, 4, 128),
}
FEW16 = {
    "four of four": ([700, 129, 128, 4, 3000, 2], [4, 3, 4, 4, 4, 4], 32, 8, 16),
    "sixteen of one": ([500, 16, 3, 1200], [16, 9, 16, 13], 2, 2, 16),
    "five of three": ([333, 64, 1000], [5, 4, 3], 12, 4, 32),
    "one of sixteen": ([900, 33, 2500], [1, 1, 1], 32, 2, 16),
    "two of eight": ([900, 33, 1], [2, 1, 2], 16, 2, 8),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name, quant", [(n, q) for n in FEW for q in (False, True)] + [(n, False) for n in FEW16])
def test_sessions_of_a_few_rows_match_64_bits(name, quant, d, dtype):
    dev = need_gpu()
    lens, new, hq, hkv, bs = {**FEW, **FEW16}[name]
    case = Case(lens, new, hq, hkv, d, bs, dtype, seed=30 + len(name), quant=quant)
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("quant, d, dtype, n_short, s_short", [(True, 128, BF, 17, 3200), (True, 64, HF, 9, 11000),
                                                              (False, 128, HF, 8, 27001), (False, 64, BF, 70, 5600)])
def test_both_kernels_in_one_call(quant, d, dtype, n_short, s_short):
    """Short sessions of 64 MB of 8-bit rows (512 MB of 16-bit ones) and more beside longer ones: the two tensor-core
    kernels share the call, each skips the other's sessions, and both leave units cut between CTAs to the join."""
    dev = need_gpu()
    from actkv_open_b200.kernels.chunk_attn import paged_chunk_attention
    from actkv_open_b200.kernels.quant_cache import (dequantize_read, paged_chunk_attention_quant, quant_row_bytes,
                                                     quantize_write)
    hq, hkv, bs = 32, 8, 16
    lens = [s_short + 7 * i for i in range(n_short)]
    new = [i % 3 for i in range(n_short)]
    for at, s, a in ((0, 1500, 300), (3, 6000, 70), (len(lens), 40, 40), (len(lens) - 1, 5, 130)):
        lens.insert(at, s)
        new.insert(at, a)
    short = sum(s for s, a in zip(lens, new) if 0 < a <= 2)
    assert short * hkv * d * 2 * (1 if quant else 2) >= (64 if quant else 512) << 20
    gen = torch.Generator(device=dev).manual_seed(31)
    table, nb = C.pages(lens, bs, torch.Generator().manual_seed(31))
    off = C.offsets(new)
    table, seq, q_off = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), off.to(dev)
    q = torch.randn(int(off[-1]), hq, d, generator=gen, device=dev).to(dtype)
    n = sum(lens)
    k, v = (torch.randn(1, n, hkv, d, generator=gen, device=dev).to(dtype) for _ in range(2))
    tok_off = C.offsets(lens).to(dev)
    if quant:
        rows = torch.full((1, 2, nb, bs, quant_row_bytes(hkv, d)), 255, dtype=torch.uint8, device=dev)
        quantize_write(k, v, tok_off, rows, table, seq)
        k, v = dequantize_read(rows, hkv, d, tok_off, table, seq, n, dtype=dtype)
        call = lambda: paged_chunk_attention_quant(q, q_off, rows[0], hkv, table, seq)                 # noqa: E731
    else:
        kv = torch.full((2, nb, bs, hkv, d), float("nan"), dtype=dtype, device=dev)
        for r, s in enumerate(lens):
            pos = torch.arange(s, device=dev)
            slot = table[r].long()[pos // bs] * bs + pos % bs
            for p, x in enumerate((k, v)):
                kv[p].view(nb * bs, hkv, d)[slot] = x[0, int(tok_off[r]):int(tok_off[r]) + s]
        call = lambda: paged_chunk_attention(q, q_off, kv, table, seq)                                 # noqa: E731
    out, lse = call()
    g = hq // hkv
    for r, (s, a) in enumerate(zip(lens, new)):
        if a == 0:
            continue
        o0, o1, t0 = int(off[r]), int(off[r + 1]), int(tok_off[r])
        kk, vv = (x[0, t0:t0 + s].double() for x in (k, v))
        qq = q[o0:o1].double().view(a, hkv, g, d)
        hide = torch.arange(s, device=dev)[None] > torch.arange(s - a, s, device=dev)[:, None]
        x = (torch.einsum("ahgd,shd->ahgs", qq, kk) * d ** -0.5).masked_fill(hide[:, None, None], -torch.inf)
        one = torch.logsumexp(x, -1)
        p = torch.where(torch.isfinite(one)[..., None], torch.exp(x - one[..., None]), torch.zeros_like(x))
        want, mag = (torch.einsum("ahgs,shd->ahgd", p, y).reshape(a, hq, d) for y in (vv, vv.abs()))
        size = (torch.einsum("ahgd,shd->ahgs", qq.abs(), kk.abs()).amax(-1) * d ** -0.5).view(a, hq)
        one = one.view(a, hq)
        tol = (2 * U[dtype] + 1e-4) * mag + (s * 2.0 ** -25 * vv.abs().amax() if dtype == HF else 0.0)
        assert ((out[o0:o1].double() - want).abs() <= tol).all(), r
        none = one == -torch.inf
        assert torch.equal(lse[o0:o1] == -torch.inf, none) and (out[o0:o1][none] == 0).all()
        assert ((lse[o0:o1].double() - one).abs()[~none] <= (2e-5 + 8e-6 * size)[~none]).all(), r
    for _ in range(3):
        assert _equal((out, lse), call())
    assert_device_clean(dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens", [500, 6000])
@pytest.mark.parametrize("new, hq, d", [(1, 8, 128), (2, 16, 64), (4, 16, 128), (4, 8, 64), (90, 8, 128), (200, 8, 64)])
def test_values_that_are_not_finite(new, hq, d, lens, dtype):
    """inf, -inf and NaN in a value of 16-bit rows, and a NaN group (scale byte 255) of 8-bit ones, at a session's start,
    in its middle and among its new tokens, in the kernels for few rows (up to 16, whole and cut between CTAs) and many:
    in that dim of the rows that see the token, and nowhere else."""
    dev = need_gpu()
    for quant in (False, True):
        case = Case([lens, 40], [new, 1], hq, 4, d, 16, dtype, seed=32, quant=quant)
        clean = case.run(dev)
        rows, head, dim, g = case.cache.clone(), 2, 37, hq // 4
        q = torch.arange(head * g, head * g + g)
        for tok in sorted({0, lens // 2 + 3, lens - new + new // 2, lens - 1}):
            at, see = int(C.slots(case.table, 0, tok, tok + 1, 16)), max(0, tok - (lens - new))
            for bad in ((float("inf"), -float("inf"), float("nan")) if not quant else (255,)):
                case.cache = rows.clone()
                dims = [dim] if not quant else list(range(32, 64))
                if quant:
                    case.cache[1, at, 4 * d + (head * d + 32) // 32] = 255
                else:
                    case.cache[1, at, head, dim] = bad
                out, lse = case.run(dev)
                assert torch.equal(lse, clean[1])
                hit = out[see:new][:, q][..., dims]
                assert torch.isnan(hit).all() if bad != bad or quant else (hit == bad).all()
                want = clean[0].clone()
                want[see:new, q[:, None], torch.tensor(dims)[None]] = hit
                assert torch.equal(torch.nan_to_num(out, nan=77.0), torch.nan_to_num(want, nan=77.0))
                assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("new", [1, 90])
def test_a_negative_length_is_an_empty_session(new, quant):
    """Its queries see nothing; the sessions beside it are as without it."""
    dev = need_gpu()
    case = Case([300, 40, 700], [new, 2, new], 8, 4, 128, 16, BF, seed=33, quant=quant)
    x = case.device(dev)
    want = case.run(dev, given={**x, "seq": torch.tensor([300, 0, 700], dtype=torch.int32, device=dev)})
    for path in ("auto", "simt"):
        base = want if path == "auto" else case.run(dev, given={**x, "seq": torch.tensor([300, 0, 700], dtype=torch.int32, device=dev)}, path=path)
        for bad in (-1, -100000, -(1 << 31) + 1000):
            got = case.run(dev, given={**x, "seq": torch.tensor([300, bad, 700], dtype=torch.int32, device=dev)}, path=path)
            assert _equal(base, got)
            assert (got[0][new:new + 2] == 0).all() and (got[1][new:new + 2] == -torch.inf).all()
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("width", [3, 8])
def test_lengths_past_the_table(width, new, quant):
    """A length that its table has no place for, up to the largest there is: flagged, the tokens past the table are
    hidden (and not walked, whatever the length), and the session beside it is as it should be."""
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    room = width * 16
    case = Case([room, 120], [new, 2], 8, 4, 128, 16, BF, seed=34, quant=quant)
    x = case.device(dev)
    x["table"] = x["table"][:, :width].contiguous()
    if width == 3:
        case.lens[1] = 40
        x["seq"][1] = 40
    for length in (room + 1, 5000, 1 << 30, (1 << 31) - 1):
        seq = x["seq"].clone()
        seq[0] = length
        first = [max(0, min(room, length - new + j + 1)) for j in range(new)]
        refs = [t.double().repeat_interleave(2, 1) for t in (case.tokens(0, 0), case.tokens(1, 0))]
        logit = torch.einsum("ahd,shd->ahs", case.q[:new].double(), refs[0]) * 128 ** -0.5
        hide = torch.arange(room)[None] >= torch.tensor(first)[:, None]
        logit = logit.masked_fill(hide[:, None], -torch.inf)
        one = torch.logsumexp(logit, -1)
        p = torch.where(torch.isfinite(one)[..., None], torch.exp(logit - one[..., None]), torch.zeros_like(logit))
        out, lse, mag, size = case.ref()
        out[:new], mag[:new] = (torch.einsum("ahs,shd->ahd", p, v) for v in (refs[1], refs[1].abs()))
        lse[:new] = one
        size[:new] = torch.einsum("ahd,shd->ahs", case.q[:new].double().abs(), refs[0].abs()).amax(-1) * 128 ** -0.5
        for path in ("auto", "simt"):
            _within(case.run(dev, given={**x, "seq": seq}, path=path), (out, lse, mag, size))
            torch.cuda.synchronize()
            assert N.read_device_status(dev) == N.DEV_BAD_INDEX
