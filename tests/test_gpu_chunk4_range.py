"""Attention over the 4-bit cache where scales are far apart: values whose size has nothing to do with their weight.

The bounds are those of test_gpu_chunk.py, with what the kernel for few rows adds.  It holds p times 2^7 in fp16, times 2^(b - E)
for a token's scale byte b in E - 7 .. E, where fp16 numbers below 2^-14 err by 2^-25 at most; m is the maximum of the logits of the
tokens that are added that way, and all others are added in 32 bits.  E rises by up to 3 before m is set anew.  A token so errs by
6 2^-25 2^-7 2^(E - 127) at most, and the token with p = 1 has a value of 4 2^(E - 10 - 127) at least among the 32 of its
group: S tokens err by S 2^-21 times what that one gives.  |out - ref| <= (2 u + 1e-4) A + S 2^-21 max of A over the group, A = sum p |v| / l; fp16: + 2^-25 for the result.  And a p of
less than 2^-126 of the largest is below what 32 bits hold as normal numbers: it may be anything down to 0, + sum of those p |v| / l."""
import math

import pytest
import torch

import chunk_cases as C
from gpu_util import assert_device_clean, need_gpu
from test_gpu_chunk import BF, HF, U
from test_gpu_chunk4 import Case4

pytestmark = pytest.mark.gpu

NEW = [1, 3, 9, 90]


def _session(lens, new, d, dtype, low, seed, hkv=2, hq=4):
    """A session whose logits (with scale 1) are 4 times dim 0 of its keys, exactly: up to 2.5 apart, those of the tokens
    in ``low`` that much lower."""
    case = Case4.__new__(Case4)
    gen = torch.Generator().manual_seed(seed)
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    case.lens, case.new, case.hq, case.hkv, case.d, case.bs, case.dtype, case.quant = [lens], [new], hq, hkv, d, 16, dtype, True
    case.table, case.nb = C.pages([lens], 16, gen)
    case.off, case.row = C.offsets([new]), quant_row_bytes(hkv, d, 4)
    case.cache = torch.full((2, case.nb * 16, case.row), 255, dtype=torch.uint8)
    case.q = torch.zeros(new, hq, d, dtype=dtype)
    case.q[..., 0] = 4
    k = torch.randn(lens, hkv, d, generator=gen)
    k[..., 0] = torch.rand(lens, hkv, generator=gen) * 0.625
    for t, drop in low.items():
        k[t] = 0                             # (the other dims of its group would not fit beside it)
        k[t, :, 0] = -drop / 4
    case.put(0, 0, k.to(dtype))
    case.v = [torch.randn(lens, hkv, d, generator=gen)]
    return case


def _reference(case, dev, scale=1.0):
    s, a, g = case.lens[0], case.new[0], case.hq // case.hkv
    k, v = (case.tokens(p, 0).double().to(dev).repeat_interleave(g, 1) for p in range(2))
    q = case.q.double().to(dev)
    x = torch.einsum("ahd,shd->ahs", q, k) * scale
    x = x.masked_fill((torch.arange(s, device=dev) > torch.arange(s - a, s, device=dev)[:, None])[:, None], -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[..., None])
    size = torch.einsum("ahd,shd->ahs", q.abs(), k.abs()).amax(-1) * scale
    tiny = torch.where(p < 2.0 ** -126 * p.amax(-1, keepdim=True), p, torch.zeros_like(p))
    mag, lost = (torch.einsum("ahs,shd->ahd", y, v.abs()) for y in (p, tiny))
    return torch.einsum("ahs,shd->ahd", p, v), lse, mag, size, lost


def _check(case, dev, got, scale=1.0):
    want, want_l, mag, size, lost = _reference(case, dev, scale)
    out, lse = (x.double() for x in got)
    group = mag.unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
    tol = (2 * U[case.dtype] + 1e-4) * mag + case.lens[0] * 2.0 ** -21 * group + lost + (2.0 ** -25 if case.dtype == HF else 0.0)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    off = (out - want).abs() - tol
    worst = int(off.argmax())
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} outputs off, one {out.flatten()[worst]:.5g} for " \
        f"{want.flatten()[worst]:.5g}, sum p |v| {mag.flatten()[worst]:.5g}"
    assert ((lse - want_l).abs() <= 2e-5 + 8e-6 * size).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", NEW)
def test_a_large_value_of_no_weight_leaves_the_others_their_share(new, d, dtype):
    """One token, 60 below all others in its logit, with values 2^spread times theirs: early in the session, in its middle,
    at its end, and among the new tokens.  Its share is e^-60 2^spread at most."""
    dev = need_gpu()
    lens = 1000
    base = 1.0 if dtype == BF else 2.0 ** -10                # (fp16 reads end at 65504)
    for spread in (6, 10, 16, 20, 24, 26, 30, 50) if dtype == BF else (6, 10, 13, 22):
        for at in ([0], [500], [lens - new], [lens - 1], [0, 33, 34, 700, 998]):
            case = _session(lens, new, d, dtype, {t: 60 for t in at}, 60 + spread)
            size = torch.full((lens, 1, 1), base)
            size[at] *= 2.0 ** spread
            case.put(1, 0, (case.v[0] * size).to(dtype))
            if spread % 4 == 2:              # ... of one head and group only
                for t in at:
                    row = case.cache[1, int(C.slots(case.table, 0, t, t + 1, 16))]
                    keep = int(row[case.scale_at(1, 1)])
                    row[case.scale_at(0, 0):case.scale_at(2, 0)] -= spread
                    row[case.scale_at(1, 1)] = keep
            _check(case, dev, case.run(dev, scale=1.0))
    assert_device_clean(dev)


@pytest.mark.parametrize("new", NEW)
def test_values_large_in_proportion_to_their_little_weight(new):
    """Values 2^n times as large on tokens whose weight is about 2^-n: each has its share of the output."""
    dev = need_gpu()
    lens = 700
    for seed, steps in enumerate(([0, 9, 18, 27], list(range(0, 64, 3)), [0] * 60 + [40], [0, 12, 0, 0, 0], [80, 0],
                                  [0] * 100 + [20] * 150)):
        shift = [steps[t % len(steps)] for t in range(lens)]
        case = _session(lens, new, 128, BF, {t: n * math.log(2) for t, n in enumerate(shift) if n}, 70 + seed)
        case.put(1, 0, (case.v[0] * torch.tensor([2.0 ** n for n in shift])[:, None, None]).to(BF))
        _check(case, dev, case.run(dev, scale=1.0))
    assert_device_clean(dev)


@pytest.mark.parametrize("new", NEW)
def test_runs_of_tokens_of_unlike_scales(new):
    """Equal weights but for the largest values': stretches, single tokens and zeros between them, up to the ends of the range."""
    dev = need_gpu()
    lens = 900
    gen = torch.Generator().manual_seed(3)
    up = lambda *runs: [x for n, k in runs for x in [k] * n]                                             # noqa: E731
    for seed, (shift, heavy) in enumerate((
            (up((300, 0), (200, -40), (400, 0)), 1000), (up((64, 100), (836, 0)), 50), (up((1, 110), (899, -60)), 0),
            (up((450, -100), (2, 100), (448, -100)), 0), ([0 if t % 2 else None for t in range(lens)], 1000),
            (torch.randint(-8, 9, (lens,), generator=gen).tolist(), 1000),
            (torch.randint(-30, 60, (lens,), generator=gen).tolist(), 5), ([None] * 100 + [-20] * 800, 1000))):
        low = {t: 120 for t, n in enumerate(shift) if n is not None and n > heavy}
        case = _session(lens, new, 128, BF, low, 80 + seed)
        size = torch.tensor([0.0 if n is None else 2.0 ** n for n in shift])
        case.put(1, 0, (case.v[0] * size[:, None, None]).to(BF))
        _check(case, dev, case.run(dev, scale=1.0))
    assert_device_clean(dev)


@pytest.mark.parametrize("new", NEW)
def test_a_dominant_token_of_small_values(new):
    """A token with nearly all the weight and values 2^-n of the others', or none: theirs count by what is left to them."""
    dev = need_gpu()
    lens = 600
    for seed, (n, at) in enumerate(((30, [0]), (30, [300]), (None, [5]), (None, [597 - new]), (60, [0, 1, 2]))):
        drop = 25 if n is None else n * math.log(2)
        case = _session(lens, new, 128, BF, {t: drop for t in range(lens) if t not in at}, 90 + seed)
        size = torch.ones(lens, 1, 1)
        size[at] = 0.0 if n is None else 2.0 ** -n
        case.put(1, 0, (case.v[0] * size).to(BF))
        _check(case, dev, case.run(dev, scale=1.0))
    assert_device_clean(dev)


def _keys(case, codes, scales):
    """The session's keys from their bytes: codes [S, Hkv * D / 2], scales [S, Hkv * D / 32]."""
    at, n = C.slots(case.table, 0, 0, case.lens[0], 16), case.hkv * case.d // 2
    case.cache[0, at, :n] = codes.to(torch.uint8)
    case.cache[0, at, n:n + case.hkv * case.d // 32] = scales.to(torch.uint8)


@pytest.mark.parametrize("path", ["auto", "simt"])
@pytest.mark.parametrize("new", NEW)
def test_the_smallest_keys_count_beside_the_largest_queries(new, path):
    """Keys of scale bytes 0 and 1 (up to 6 2^-126) and queries of 2^123: logits of the order of 1, wherever the token stands."""
    dev = need_gpu()
    lens = 300
    for d in (64, 128):
        case = _session(lens, new, d, BF, {}, 50)
        case.put(1, 0, case.v[0].to(BF))
        gen = torch.Generator().manual_seed(51)
        _keys(case, torch.randint(0, 256, (lens, d), generator=gen), torch.randint(0, 2, (lens, d // 16), generator=gen))
        case.q = ((torch.randint(0, 2, (new, 4, d), generator=gen) * 2 - 1) * 2.0 ** 123).to(BF)
        _check(case, dev, case.run(dev, scale=1.0, path=path))
    assert_device_clean(dev)


@pytest.mark.parametrize("path", ["auto", "simt"])
@pytest.mark.parametrize("new", NEW)
def test_large_keys_beside_queries_of_zero(new, path):
    """Dims where the queries are 0 and some keys up to 6 2^123, beside dims of queries of 2^100 and keys of 2^-100: those
    alone make the logits."""
    dev = need_gpu()
    lens = 300
    for d in (64, 128):
        case = _session(lens, new, d, BF, {}, 52)
        case.put(1, 0, case.v[0].to(BF))
        gen = torch.Generator().manual_seed(53)
        scales = torch.full((lens, 2, d // 32), 27)
        scales[::7, :, 1] = 250
        _keys(case, torch.randint(0, 256, (lens, d), generator=gen), scales.flatten(1))
        q = torch.randn(new, 4, d, generator=gen) * 2.0 ** 98
        q[..., 32:64] = 0
        case.q = q.to(BF)
        _check(case, dev, case.run(dev, scale=0.25, path=path), 0.25)
    assert_device_clean(dev)


@pytest.mark.parametrize("path", ["auto", "simt"])
@pytest.mark.parametrize("new", NEW)
def test_queries_and_keys_whose_groups_are_far_apart(new, path):
    """Groups of 32 dims in which queries are 2^n times as large and keys 2^-n times: each has its share in the logits."""
    dev = need_gpu()
    lens = 300
    for seed, shift in enumerate(([0, 40], [20, -20, 0, 10], [0, 13, 26, -14], [100, -100], [-60, 0, 60, None], [12, 0], [29, 0])):
        d = 32 * len(shift)
        case = _session(lens, new, d, BF, {}, 54 + seed)
        case.put(1, 0, case.v[0].to(BF))
        gen = torch.Generator().manual_seed(60 + seed)
        scales = torch.tensor([125 - (n or 0) for n in shift]).expand(lens, 2, -1).clone()
        scales += torch.randint(0, 2, scales.shape, generator=gen)
        _keys(case, torch.randint(0, 256, (lens, d), generator=gen), scales.flatten(1))
        size = torch.tensor([0.0 if n is None else 2.0 ** n for n in shift]).repeat_interleave(32)
        case.q = (torch.randn(new, 4, d, generator=gen) * size).to(BF)
        case.q[:, 1::2] *= 0.5
        case.q[new // 2, 2] = 0
        _check(case, dev, case.run(dev, scale=d ** -0.5, path=path), d ** -0.5)
    assert_device_clean(dev)


def test_a_group_of_nan_holds_up_nobody():
    """Two sessions of 60000 tokens in one call, a NaN group in the first: the other's results are as without it, and the call
    takes about as long (its tokens are looked at once more at the end of the unit, 32 at a time; it took six times as long
    where one lane looked at all, in every later unit too)."""
    dev = need_gpu()
    from actkv_open_b200.kernels.chunk_attn import chunk_workspace
    from actkv_open_b200.kernels.quant_cache import paged_chunk_attention_quant, quant_row_bytes
    hkv, d, s, r = 8, 128, 60000, 2
    nb = r * s // 16
    gen = torch.Generator(device=dev).manual_seed(1)
    rows = torch.randint(0, 256, (2, nb, 16, quant_row_bytes(hkv, d, 4)), generator=gen, device=dev, dtype=torch.uint8)
    rows[..., hkv * d // 2:] = torch.randint(124, 127, rows[..., hkv * d // 2:].shape, generator=gen, device=dev, dtype=torch.uint8)
    table = torch.arange(nb, dtype=torch.int32, device=dev).view(r, -1)
    seq, off = torch.full((r,), s, dtype=torch.int32, device=dev), torch.arange(r + 1, dtype=torch.int32, device=dev) * 2
    q = torch.randn(2 * r, 32, d, generator=gen, device=dev).bfloat16()
    ws = chunk_workspace(dev)

    def timed():
        best = math.inf
        for _ in range(8):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            got = paged_chunk_attention_quant(q, off, rows, hkv, table, seq, workspace=ws, bits=4)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return got, best

    clean, before = timed()
    rows[1, 3, 5, hkv * d // 2 + 4 * 2 + 1] = 255          # head 2, group 1, token 53 of the first session
    got, after = timed()
    bad = torch.zeros(2 * r, 32, d, dtype=torch.bool, device=dev)
    bad[:2, 8:12, 32:64] = True
    assert torch.isnan(got[0][bad]).all() and torch.equal(got[0][~bad], clean[0][~bad]) and torch.equal(got[1], clean[1])
    assert after < 3 * before, f"{before * 1e3:.0f} us without, {after * 1e3:.0f} us with one group of NaN"
    assert_device_clean(dev)


@pytest.mark.parametrize("new", NEW)
def test_sessions_that_begin_with_zeros(new):
    """The first tokens have nearly all the weight and zeros for values, after sessions of ordinary and of large ones in the
    same call: what the others have is theirs."""
    dev = need_gpu()
    lens, first = 200, 64
    for drop, shift in ((25, 0), (20, 60), (20, -60)):
        case = _session(lens, new, 128, BF, {t: drop for t in range(first, lens)}, 95)
        size = torch.full((lens, 1, 1), 2.0 ** shift)
        size[:first] = 0
        case.put(1, 0, (case.v[0] * size).to(BF))
        alone = case.run(dev, scale=1.0)
        _check(case, dev, alone)
        # the same session forty times, every other one with ordinary values at its start
        x = case.device(dev)
        r = 40
        rows = torch.cat([x["cache"]] * 2, 1)
        at = C.slots(case.table, 0, 0, first, 16).to(dev)
        rows[1].flatten(0, 1)[case.nb * 16 + at] = rows[1].flatten(0, 1)[C.slots(case.table, 0, lens - first, lens, 16).to(dev)]
        table = torch.cat([x["table"] + case.nb, x["table"]]).repeat(r // 2, 1)
        out, lse = case.run(dev, scale=1.0, given=dict(
            q=case.q.to(dev).repeat(r, 1, 1), q_off=C.offsets([new] * r).to(dev), cache=rows, table=table.contiguous(),
            seq=torch.full((r,), lens, dtype=torch.int32, device=dev)))
        for i in range(1, r, 2):
            _check(case, dev, (out[i * new:(i + 1) * new], lse[i * new:(i + 1) * new]))
    assert_device_clean(dev)
