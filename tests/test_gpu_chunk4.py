"""Chunk attention over the 4-bit cache against a 64-bit statement of the formula, on the tensor cores and on CUDA
cores.  Bounds as derived in test_gpu_chunk.py; where the kernel for few rows holds p in fp16 (times 2^7, times a
power of two of at most 1 for the token's scale) instead of the output's type, p errs by less."""
import math

import pytest
import torch

import chunk_cases as C
import quant4_cases as Q
from gpu_util import assert_device_clean, need_gpu
from test_gpu_chunk import BF, FP, HF, SHAPES, U, Case, _equal
from test_gpu_chunk_edges import FEW, _holes_ref, _within

pytestmark = pytest.mark.gpu


class Case4(Case):
    """``Case`` over rows of 4 bits (NaN in every slot that holds no token)."""

    def __init__(self, lens, new, hq, hkv, d, bs, dtype, seed=0, gain=1.0):
        super().__init__(lens, new, hq, hkv, d, bs, dtype, seed=seed, gain=gain)
        from actkv_open_b200.kernels.quant_cache import quant_row_bytes
        self.quant, self.row = True, quant_row_bytes(hkv, d, 4)
        self.cache = torch.full((2, self.nb * bs, self.row), 255, dtype=torch.uint8)
        for r, s in enumerate(lens):
            for p, x in enumerate((self.k[r], self.v[r])):
                self.put(p, r, x)

    def put(self, p, r, x):
        self.cache[p, C.slots(self.table, r, 0, self.lens[r], self.bs)] = Q.pack_rows(x, self.row)

    def tokens(self, p, r):
        return Q.unpack_rows(self.cache[p, C.slots(self.table, r, 0, self.lens[r], self.bs)], self.hkv, self.d)

    def scale_at(self, head, group):
        """Where a head's scale bytes are in a row."""
        return self.hkv * self.d // 2 + head * (self.d // 32) + group

    def run(self, dev, **kw):
        from actkv_open_b200.kernels.quant_cache import paged_chunk_attention_quant
        given = kw.pop("given", {})
        x = given if len(given) == 5 else {**self.device(dev), **given}
        return paged_chunk_attention_quant(x["q"], x["q_off"], x["cache"], self.hkv, x["table"], x["seq"], bits=4, **kw)


@pytest.mark.parametrize("name", [n for n in SHAPES if SHAPES[n][4] in (64, 96, 128)])
def test_matches_64_bits(name):
    dev = need_gpu()
    case = Case4(*SHAPES[name], seed=len(name))
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("name", ["drafted", "chunk", "mixed with idle and empty sessions", "d 64"])
def test_cuda_core_path(name):
    dev = need_gpu()
    case = Case4(*SHAPES[name], seed=3)
    case.check(case.run(dev, path="simt"))
    assert_device_clean(dev)


GROUPS = {   # lens, new, hq, hkv, block size: 9 to 32 rows per KV head, in groups of up to 8
    "four of four": ([700, 129, 128, 4, 3000, 2], [4, 3, 4, 4, 4, 4], 32, 8, 16),
    "sixteen of one": ([500, 16, 3, 1200], [16, 9, 16, 13], 2, 2, 16),
    "ten of three": ([333, 64, 1000], [10, 4, 3], 12, 4, 32),
    "four of eight": ([900, 33, 2, 2500], [4, 3, 4, 2], 32, 4, 16),
    "six of five, one KV head": ([900, 33], [6, 5], 5, 1, 8),
    "thirty-two of one, and longer": ([2000, 31, 400, 64], [32, 32, 33, 1], 8, 8, 64),
    "seven of four, many": ([40 + 13 * i for i in range(40)], [i % 8 for i in range(40)], 8, 2, 16),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", GROUPS)
def test_sessions_of_several_groups_of_rows_match_64_bits(name, d, dtype):
    dev = need_gpu()
    lens, new, hq, hkv, bs = GROUPS[name]
    case = Case4(lens, new, hq, hkv, d, bs, dtype, seed=50 + len(name))
    x = case.device(dev)
    first = case.run(dev, given=x)
    case.check(first)
    assert _equal(first, case.run(dev, given=x))
    assert_device_clean(dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", FEW)
def test_sessions_of_a_few_rows_match_64_bits(name, d, dtype):
    dev = need_gpu()
    lens, new, hq, hkv, bs = FEW[name]
    case = Case4(lens, new, hq, hkv, d, bs, dtype, seed=30 + len(name))
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HF)])
def test_both_kernels_in_one_call(d, dtype):
    """Short sessions of 32 MB of rows and more, of one and of several groups of rows, beside longer ones."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, paged_chunk_attention_quant, quant_row_bytes, quantize_write
    hq, hkv, bs = 32, 8, 16
    lens = [6400 * 128 // d + 7 * i for i in range(9)]
    new = [(0, 1, 2, 5, 8)[i % 5] for i in range(9)]
    for at, s, a in ((0, 1500, 300), (3, 6000, 70), (len(lens), 40, 40), (len(lens) - 1, 5, 130)):
        lens.insert(at, s)
        new.insert(at, a)
    assert sum(s for s, a in zip(lens, new) if 0 < a <= 8) * hkv * d >= 32 << 20
    gen = torch.Generator(device=dev).manual_seed(31)
    table, nb = C.pages(lens, bs, torch.Generator().manual_seed(31))
    off = C.offsets(new)
    table, seq, q_off, tok = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), off.to(dev), C.offsets(lens).to(dev)
    q = torch.randn(int(off[-1]), hq, d, generator=gen, device=dev).to(dtype)
    n = sum(lens)
    k, v = (torch.randn(1, n, hkv, d, generator=gen, device=dev).to(dtype) for _ in range(2))
    rows = torch.full((1, 2, nb, bs, quant_row_bytes(hkv, d, 4)), 255, dtype=torch.uint8, device=dev)
    quantize_write(k, v, tok, rows, table, seq, bits=4)
    k, v = dequantize_read(rows, hkv, d, tok, table, seq, n, dtype=dtype, bits=4)
    call = lambda: paged_chunk_attention_quant(q, q_off, rows[0], hkv, table, seq, bits=4)             # noqa: E731
    out, lse = call()
    g = hq // hkv
    for r, (s, a) in enumerate(zip(lens, new)):
        if a == 0:
            continue
        o0, o1, t0 = int(off[r]), int(off[r + 1]), int(tok[r])
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


def test_many_sessions_and_long_ragged_ones():
    dev = need_gpu()
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(1, 300, (70,), generator=g).tolist() + [9000, 4097]
    new = [min(s, int(n)) for s, n in zip(lens, torch.randint(0, 5, (72,), generator=g))]
    new[-1] = 70
    case = Case4(lens, new, 8, 2, 128, 16, BF, seed=4)
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("new", [(130, 1), (2, 1)])
@pytest.mark.parametrize("gain", [0.0, 6.0])
def test_flat_and_peaked_logits(gain, new):
    dev = need_gpu()
    case = Case4([1000, 300], list(new), 8, 2, 128, 16, BF, seed=5, gain=gain)
    at = C.slots(case.table, 0, 0, 1000, 16)
    case.cache[:, at] = case.cache[:, at[torch.argsort(case.k[0][:, 0, 0].float())]]
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 9, 90])
def test_scales_far_apart(new, d, dtype):
    """Tokens, groups and heads whose scales differ by up to 2^16, the largest values on tokens of little weight and on
    the newest (which some rows do not see): every value counts by its weight, in every row."""
    dev = need_gpu()
    lens = [900, 70]
    case = Case4(lens, [new, 1], 8, 4, d, 16, dtype, seed=41)
    gen = torch.Generator().manual_seed(42)
    for r, s in enumerate(lens):
        size = 2.0 ** torch.randint(-8, 9, (s, 4, d // 32, 1), generator=gen)
        v = (case.v[r].float().view(s, 4, -1, 32) * size).view(s, 4, d).to(dtype)
        size = 2.0 ** torch.randint(-3, 2, (s, 4, d // 32, 1), generator=gen)
        k = (case.k[r].float().view(s, 4, -1, 32) * size).view(s, 4, d).to(dtype)
        case.put(0, r, k)
        case.put(1, r, v)
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("new", [2, 4, 11, 90])
@pytest.mark.parametrize("lens", [500, 6000])
@pytest.mark.parametrize("byte", [150, 200, 252])
def test_large_hidden_values_reach_only_the_rows_that_see_them(byte, lens, new):
    """The last token's values 2^(byte - 126) times the others': the rows before it are as without it, bit for bit."""
    dev = need_gpu()
    case = Case4([lens, 40], [new, 1], 8, 4, 128, 16, BF, seed=43)
    clean = case.run(dev)
    at = int(C.slots(case.table, 0, lens - 1, lens, 16))
    case.cache[1, at, case.scale_at(0, 0):case.scale_at(4, 0)] = byte
    got = case.run(dev)
    rows = list(range(new - 1)) + [new]
    assert _equal([x[rows] for x in got], [x[rows] for x in clean]) and torch.equal(got[1], clean[1])
    want, _, mag, _ = case.ref()
    assert ((got[0][new - 1].cpu().double() - want[new - 1]).abs() <= (2 * U[BF] + 1e-4) * mag[new - 1]).all()
    # ... and keys: 2^60 times the others'; the row that sees them sees nothing else (the kernel for many rows tells logits
    # apart up to 2^24, as over the other caches: there that row's own result says nothing)
    case.cache[1, at, case.scale_at(0, 0):case.scale_at(4, 0)] = 126
    case.cache[0, at, case.scale_at(0, 0):case.scale_at(4, 0)] = min(byte, 186)
    got = case.run(dev)
    assert _equal([x[rows] for x in got], [x[rows] for x in clean])
    if new < 16:
        assert not torch.isnan(got[0]).any() and not torch.isnan(got[1]).any()
        one = got[0][new - 1].cpu().double()
        logits = case.q[new - 1].double().view(4, 2, 1, 128) * case.tokens(0, 0)[-1].view(4, 1, 1, 128)
        alone = logits.sum(-1).view(8) > 0               # its logit is the largest, by far
        value = case.tokens(1, 0)[-1].repeat_interleave(2, 0)
        assert alone.any() and torch.equal(one[alone], value[alone].to(BF).double())
    assert_device_clean(dev)


@pytest.mark.parametrize("path", ["auto", "simt"])
@pytest.mark.parametrize("new", [1, 3, 9, 90])
def test_hidden_tokens_do_not_reach_a_query(path, new):
    """NaN groups (scale bytes 253 to 255) among keys and values, at a session's start, in its middle and among its new
    tokens: a value makes its group's dims NaN in the rows that see it, a key the whole row of its head, and nothing
    else changes."""
    dev = need_gpu()
    for lens, d, dtype, hq in ((500, 128, BF, 8), (500, 64, HF, 16), (6000, 128, HF, 8), (6000, 64, BF, 8)):
        case = Case4([lens, 40], [new, 1], hq, 4, d, 16, dtype, seed=44)
        clean = case.run(dev, path=path)
        rows, head, group, g = case.cache.clone(), 2, 1, hq // 4
        q = torch.arange(head * g, head * g + g, device=dev)
        others = [h for h in range(hq) if h // g != head]
        for tok in sorted({0, lens // 2 + 3, lens - new + new // 2, lens - 1}):
            at, see = int(C.slots(case.table, 0, tok, tok + 1, 16)), max(0, tok - (lens - new))
            for plane, byte in ((1, 255), (1, 253), (0, 255), (0, 254)):
                case.cache = rows.clone()
                case.cache[plane, at, case.scale_at(head, group)] = byte
                out, lse = case.run(dev, path=path)
                assert torch.equal(out[:, others], clean[0][:, others]) and torch.equal(lse[:, others], clean[1][:, others])
                assert _equal((out[:see], lse[:see]), [x[:see] for x in clean])
                assert _equal((out[new:], lse[new:]), [x[new:] for x in clean])
                if plane == 0:
                    assert torch.isnan(out[see:new, q]).all() and torch.isnan(lse[see:new, q]).all()
                else:
                    dims = list(range(32 * group, 32 * group + 32))
                    rest = [x for x in range(d) if x not in dims]
                    assert torch.isnan(out[see:new][:, q][..., dims]).all() and torch.equal(lse, clean[1])
                    assert torch.equal(out[:, q][..., rest], clean[0][:, q][..., rest])
    assert_device_clean(dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new, path", [(1, "auto"), (20, "auto"), (1, "simt")])
def test_every_scale_byte_is_attended_as_it_is_read_back(new, path, d, dtype):
    """One token per session: with a zero key the output is its value row bit for bit, and with one-hot queries the lse
    is a dim of its key.  Scale bytes 0 to 252 for the values, and for keys those of logits up to 2^24."""
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quant_row_bytes
    hkv, r = 2, 256
    gen = torch.Generator().manual_seed(26)
    codes = torch.randint(0, 256, (r, hkv * d // 2), generator=gen).to(torch.uint8)
    scale = torch.randint(0, 253, (r, hkv, d // 32), generator=gen)
    scale[:253, 0, 0] = torch.arange(253)
    scale[:60, 1, 0] = torch.arange(90, 150)
    last = torch.arange(r, device=dev) * new + new - 1
    for plane in (1, 0):
        case = Case4.__new__(Case4)
        case.lens, case.new, case.hq, case.hkv, case.d, case.bs, case.dtype, case.quant = [1] * r, [new] * r, 2 * hkv, hkv, d, 16, dtype, True
        case.table, case.nb = torch.arange(r, dtype=torch.int32)[:, None], r
        case.off = torch.arange(r + 1, dtype=torch.int32) * new
        case.row = quant_row_bytes(hkv, d, 4)
        case.cache = torch.full((2, r, 16, case.row), 255, dtype=torch.uint8)
        case.cache[:, :, 0] = 0
        case.cache[plane, :, 0, :hkv * d // 2] = codes
        most = 252 if plane or dtype == HF else 148
        case.cache[plane, :, 0, hkv * d // 2:hkv * (d // 2 + d // 32)] = scale.clamp(max=most).reshape(r, -1).to(torch.uint8)
        hot = (torch.arange(r * new)[:, None] * 7 + torch.arange(2 * hkv)[None] * 3) % d
        case.q = torch.nn.functional.one_hot(hot, d).to(dtype)
        x = case.device(dev)
        off = torch.arange(r + 1, dtype=torch.int32, device=dev)
        back = dequantize_read(x["cache"][None], hkv, d, off, x["table"], x["seq"], r, dtype=dtype, bits=4)[plane][0]
        out, lse = case.run(dev, given=x, path=path, scale=1.0)
        if plane:
            assert torch.equal(out[last], back.repeat_interleave(2, 1)) and (lse[last] == 0).all()
        else:
            want = back.repeat_interleave(2, 1).gather(2, hot.to(dev)[last][..., None])[..., 0].double()
            assert ((lse[last].double() - want).abs() <= 1e-6 * want.abs()).all() and (out[last] == 0).all()
    assert_device_clean(dev)


@pytest.mark.parametrize("new", [1, 3, 13, 90, 200])
def test_fp16_keeps_what_a_dominant_token_leaves(new):
    """As over the other caches: one token 17.4 above all others, with a zero value; the 2000 others have p = 2^-25.1."""
    dev = need_gpu()
    s = 2000
    case = Case4([s], [new], 4, 2, 128, 16, HF, seed=29)
    case.q.zero_()
    case.q[..., 0] = 17.4 / 24
    k, v = torch.zeros(s, 2, 128, dtype=HF), torch.ones(s, 2, 128, dtype=HF)
    k[0, :, 0], v[0] = 24, 0                             # 24 = 6 * 2^2 is exact in 4 bits too
    case.put(0, 0, k)
    case.put(1, 0, v)
    out, lse = (x.cpu().double() for x in case.run(dev, scale=1.0))
    want, want_l, mag, size = case.ref(1.0)
    assert (want < 1e-4).all() and (want > 2e-5).all()
    assert ((out - want).abs() <= (2 * U[HF] + 1e-4) * mag + s * 2.0 ** -32 + 2.0 ** -25).all()
    assert ((lse - want_l).abs() <= 2e-5 + 8e-6 * size).all()
    assert_device_clean(dev)


@pytest.mark.parametrize("lens, new, bs, d", [([500], [1], 16, 128), ([500], [3], 16, 64), ([500, 300], [90, 2], 16, 128),
                                              ([700, 129], [300, 33], 64, 64), ([9000], [2], 16, 128), ([900], [140], 256, 128),
                                              ([500, 90], [15, 9], 16, 128)])
def test_tokens_of_blocks_outside_the_cache_are_hidden(lens, new, bs, d):
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    case = Case4(lens, new, 8, 4, d, bs, BF, seed=25)
    x = case.device(dev)
    x["cache"] = torch.cat([torch.full_like(x["cache"][:, :1], 255), x["cache"]], 1)
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
                table[0, b] = (-1 if b % 3 else -(1 << 31)) if b % 2 else case.nb + 1 + b
                gone[0][b * bs:(b + 1) * bs] = True
        ref = _holes_ref(case, gone)
        for path in ("auto", "simt"):
            _within(case.run(dev, given={**x, "table": table}, path=path), ref)
            torch.cuda.synchronize()
            assert N.read_device_status(dev) == N.DEV_BAD_INDEX


@pytest.mark.parametrize("path", ["auto", "simt"])
@pytest.mark.parametrize("new, bad", [((2, 3, 2), (0, 2, 9, 9)), ((2, 90, 5), (0, 2, 92, 300)),
                                      ((4, 80, 5), (-3, 4, 84, 89)), ((2, 3, 2), (0, 2, 5, 1 << 30))])
def test_sessions_whose_offsets_leave_the_rows_are_left_alone(new, bad, path):
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    case = Case4([500, 300, 40], list(new), 8, 2, 128, 16, BF, seed=22)
    t = sum(new)
    room = torch.full((t + 400, 8, 128), 3.0, dtype=BF, device=dev), torch.full((t + 400, 8), 3.0, device=dev)
    case.run(dev, given=dict(q_off=torch.tensor(bad, dtype=torch.int32, device=dev)), path=path, out=room[0][200:200 + t],
             lse=room[1][200:200 + t])
    torch.cuda.synchronize()
    assert N.read_device_status(dev) == N.DEV_BAD_INDEX
    written = torch.zeros(t + 400, dtype=torch.bool, device=dev)
    for a, b in zip(bad, bad[1:]):
        if 0 <= a < b <= t:
            written[200 + a:200 + b] = True
    assert (room[0][~written] == 3).all() and (room[1][~written] == 3).all()


@pytest.mark.parametrize("d", [64, 128])
def test_units_that_see_nothing_among_units_that_do(d):
    dev = need_gpu()
    case = Case4([10, 700, 0, 421] * 4, [1000, 150, 333, 131] * 4, 8, 2, d, 16, BF, seed=21)
    x = case.device(dev)
    first = case.run(dev, given=x)
    case.check(first)
    for _ in range(3):
        assert _equal(first, case.run(dev, given=x))
    assert_device_clean(dev)


@pytest.mark.parametrize("new", [1, 3, 12, 90])
def test_negative_lengths_and_lengths_past_the_table(new):
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    case = Case4([300, 40, 700], [new, 2, new], 8, 4, 128, 16, BF, seed=33)
    x = case.device(dev)
    seq = lambda *s: torch.tensor(s, dtype=torch.int32, device=dev)                                    # noqa: E731
    want = case.run(dev, given={**x, "seq": seq(300, 0, 700)})
    for bad in (-1, -(1 << 31) + 1000):
        got = case.run(dev, given={**x, "seq": seq(300, bad, 700)})
        assert _equal(want, got) and (got[0][new:new + 2] == 0).all() and (got[1][new:new + 2] == -math.inf).all()
    assert_device_clean(dev)
    keep = x["table"].shape[1]
    for length in (keep * 16 + 1, 1 << 30, (1 << 31) - 1):
        got = case.run(dev, given={**x, "seq": seq(300, 40, length)})
        assert _equal([y[:new + 2] for y in got], [y[:new + 2] for y in case.run(dev, given=x)])
        assert N.read_device_status(dev) & N.DEV_BAD_INDEX


def test_strided_inputs_given_outputs_and_other_layouts():
    dev = need_gpu()
    from actkv_open_b200.kernels.chunk_attn import chunk_workspace
    ws = chunk_workspace(dev)
    for lens, new, seed in (([700, 40], [260, 3], 1), ([90], [1], 2), ([700, 40], [2, 3], 3)):
        case = Case4(lens, new, 8, 2, 128, 16, BF, seed=seed)
        t = case.q.shape[0]
        fused = torch.randn(t, 12, 128).to(BF).to(dev)
        fused[:, :8] = case.q.to(dev)
        stack = torch.zeros(3, 2, case.nb, 16, case.row, dtype=torch.uint8, device=dev)
        stack[1] = case.cache.view(2, case.nb, 16, case.row).to(dev)
        table = torch.full((len(lens), case.table.shape[1] + 5), -1, dtype=torch.int32, device=dev)
        table[:, :case.table.shape[1]] = case.table.to(dev)
        out = torch.full((t, 9, 160), 3.0, dtype=BF, device=dev)
        lse = torch.full((t, 10), 3.0, device=dev)
        got = case.run(dev, given=dict(q=fused[:, :8], cache=stack[1], table=table), out=out[:, :8, :128], lse=lse[:, :8],
                       workspace=ws, scale=0.2)
        case.check(got, scale=0.2)
        assert (out[:, 8] == 3).all() and (out[:, :, 128:] == 3).all() and (lse[:, 8:] == 3).all()
        # rows off 16 bytes: the CUDA cores
        odd = torch.zeros(2, case.nb, 16, case.row + 5, dtype=torch.uint8, device=dev)[..., 3:case.row + 3]
        odd.copy_(case.device(dev)["cache"])
        case.check(case.run(dev, given=dict(cache=odd)))
        with pytest.raises(NotImplementedError):
            case.run(dev, given=dict(cache=odd), path="tcgen05")
    assert_device_clean(dev)


@pytest.mark.parametrize("new", [[2, 1], [70, 1]])
def test_planes_past_32_bit_offsets(new):
    dev = need_gpu()
    first = (1 << 32) // (16 * 544) + 64
    case = Case4([500, 60], new, 8, 8, 128, 16, BF, seed=10)
    x = case.device(dev)
    big = torch.zeros((2, first + case.nb) + x["cache"].shape[2:], dtype=torch.uint8, device=dev)
    big[:, first:] = x["cache"]
    case.check(case.run(dev, given=dict(cache=big, table=x["table"] + first)))
    assert_device_clean(dev)


def test_other_streams_repeats_and_graphs_are_bitwise_equal():
    dev = need_gpu()
    from actkv_open_b200.kernels.chunk_attn import chunk_workspace
    case = Case4([3001, 500, 40], [1, 300, 5], 32, 8, 128, 16, BF, seed=11)
    x = case.device(dev)
    want = case.run(dev, given=x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [case.run(dev, given=x) for _ in range(3)]
    side.synchronize()
    assert all(_equal(want, g) for g in got)
    graph = torch.cuda.CUDAGraph()
    ws = chunk_workspace(dev)
    out, lse = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    with torch.cuda.graph(graph):
        case.run(dev, given=x, out=out, lse=lse, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert _equal(want, (out, lse))
    assert_device_clean(dev)


def test_refusals():
    dev = need_gpu()
    case = Case4([50], [3], 8, 2, 128, 16, BF)
    x = case.device(dev)
    with pytest.raises(AssertionError, match="short"):
        case.run(dev, given=dict(cache=x["cache"][..., :135]))
    with pytest.raises(AssertionError):
        case.run(dev, given=dict(cache=x["cache"].view(torch.int8)))
    with pytest.raises(RuntimeError, match="CUDA"):
        case.run(dev, given=dict(q=case.q))
    fp = Case4([50], [3], 8, 2, 128, 16, FP)
    with pytest.raises(NotImplementedError):
        fp.run(dev, path="tcgen05")
    fp.check(fp.run(dev))
    assert_device_clean(dev)
