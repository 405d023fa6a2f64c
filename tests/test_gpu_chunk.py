"""Chunk attention over a paged cache (paged_chunk_attention, paged_chunk_attention_quant) against a
64-bit statement of the formula, on the tensor cores and on CUDA cores.

The bounds.  Let u be the output type's unit roundoff (half a unit in the last place of 1.0: 2^-8 for
bf16's 8-bit significand, 2^-11 for fp16's 11 bits) and A = sum p |v| / l of an output, |out| <= A.  p is rounded to that type before it multiplies v (u A at
most over the sum) and the result once more (u A); products and sums are 32-bit, logits err by at most
~D 2^-24 sum |q k| scale and ex2 by 2^-22, well under 1e-4 relative of p for these inputs:
|out - ref| <= (2 u + 1e-4) A.  fp16 p below 2^-14 err by 2^-25 absolutely: + S 2^-25 max|v|.  fp32
rows keep p in 32 bits: 2e-5 A.  lse: 2e-5 + 8e-6 max scale sum |q k| (D 2^-24 = 7.6e-6)."""
import math

import pytest
import torch

import chunk_cases as C
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    """A paged cache on the CPU (NaN in every slot that holds no token) with the queries of a call."""

    def __init__(self, lens, new, hq, hkv, d, bs, dtype, seed=0, quant=False, fill=math.nan, gain=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.hq, self.hkv, self.d, self.bs, self.dtype, self.quant = lens, new, hq, hkv, d, bs, dtype, quant
        self.table, self.nb = C.pages(lens, bs, gen)
        self.off = C.offsets(new)
        self.q = (torch.randn(int(self.off[-1]), hq, d, generator=gen) * gain).to(dtype)
        self.k = [torch.randn(s, hkv, d, generator=gen).to(dtype) for s in lens]
        self.v = [torch.randn(s, hkv, d, generator=gen).to(dtype) for s in lens]
        if quant:
            self.row = -(-hkv * (d + d // 32) // 64) * 64
            self.cache = torch.full((2, self.nb * bs, self.row), 255, dtype=torch.uint8)     # NaN values, NaN scales
        else:
            self.cache = torch.full((2, self.nb * bs, hkv, d), fill, dtype=dtype)
        for r, s in enumerate(lens):
            for p, x in enumerate((self.k[r], self.v[r])):
                at = C.slots(self.table, r, 0, s, bs)
                self.cache[p, at] = C.pack_rows(x, self.row) if quant else x

    def tokens(self, p, r):
        at = C.slots(self.table, r, 0, self.lens[r], self.bs)
        x = self.cache[p, at]
        return C.unpack_rows(x, self.hkv, self.d) if self.quant else x

    def device(self, dev):
        shape = (2, self.nb, self.bs, self.row) if self.quant else (2, self.nb, self.bs, self.hkv, self.d)
        return dict(q=self.q.to(dev), q_off=self.off.to(dev), cache=self.cache.view(shape).to(dev),
                    table=self.table.to(dev), seq=torch.tensor(self.lens, dtype=torch.int32, device=dev))

    def run(self, dev, **kw):
        from actkv_open_b200.kernels.chunk_attn import paged_chunk_attention
        from actkv_open_b200.kernels.quant_cache import paged_chunk_attention_quant
        given = kw.pop("given", {})
        x = given if len(given) == 5 else {**self.device(dev), **given}
        if self.quant:
            return paged_chunk_attention_quant(x["q"], x["q_off"], x["cache"], self.hkv, x["table"], x["seq"], **kw)
        return paged_chunk_attention(x["q"], x["q_off"], x["cache"], x["table"], x["seq"], **kw)

    def ref(self, scale=None):
        return C.attention_ref(self.q, self.off, lambda r: self.tokens(0, r), lambda r: self.tokens(1, r), self.lens,
                               self.d ** -0.5 if scale is None else scale)

    def check(self, got, scale=None):
        out, lse = (x.cpu().double() for x in got)
        want, want_l, mag, size = self.ref(scale)
        assert not torch.isnan(out).any() and not torch.isnan(lse).any()
        if self.dtype == torch.float32:
            tol = 2e-5 * mag + 1e-30
        else:
            tol = (2 * U[self.dtype] + 1e-4) * mag
            if self.dtype == torch.float16:
                vmax = max([float(self.tokens(1, r).abs().max()) for r, s in enumerate(self.lens) if s] or [0.0])
                tol = tol + max(self.lens) * 2.0 ** -25 * vmax
        bad = (out - want).abs() > tol
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, first {bad.nonzero()[0].tolist()}: " \
            f"{out[tuple(bad.nonzero()[0])]:.6g} for {want[tuple(bad.nonzero()[0])]:.6g}"
        empty = want_l == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert (out[empty] == 0).all()
        off = (lse - want_l).abs()[~empty] - (2e-5 + 8e-6 * size[~empty])
        assert (off <= 0).all(), f"lse off by {(lse - want_l).abs()[~empty].max():.3g}"


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

# lens, new, hq, hkv, d, bs, dtype
SHAPES = {
    "one token": ([300], [1], 32, 8, 128, 16, BF),
    "length one": ([1, 1], [1, 1], 8, 2, 128, 16, BF),
    "decode batch": ([700, 129, 128, 127, 1, 2000], [1] * 6, 32, 8, 128, 16, BF),
    "drafted": ([513, 77, 1500], [5, 3, 7], 32, 8, 128, 16, BF),
    "chunk": ([700], [300], 8, 2, 128, 16, BF),
    "prompt": ([385], [385], 4, 1, 128, 16, BF),
    "two row tiles, odd end": ([421], [131], 16, 4, 128, 16, BF),
    "mixed with idle and empty sessions": ([500, 40, 0, 900, 64], [200, 0, 0, 1, 64], 16, 4, 128, 16, BF),
    "more queries than tokens": ([5, 130, 300], [9, 140, 2], 8, 2, 128, 16, BF),
    "fp16": ([600, 33], [150, 33], 16, 4, 128, 16, HF),
    "d 64": ([600, 257, 3], [140, 1, 3], 16, 4, 64, 32, BF),
    "d 64 fp16, group of 3": ([400, 90], [111, 17], 24, 8, 64, 32, HF),
    "group of 5": ([333], [60], 10, 2, 128, 16, BF),
    "group of 16": ([333, 50], [60, 1], 32, 2, 128, 16, BF),
    "group of 48, one KV head": ([200], [20], 48, 1, 128, 16, BF),
    "no grouping": ([260, 10], [130, 1], 4, 4, 128, 16, BF),
    "blocks of 8": ([200, 131], [60, 2], 8, 2, 128, 8, BF),
    "blocks of 64": ([200, 131], [60, 2], 8, 2, 128, 64, BF),
    "blocks of 128": ([500, 131], [60, 2], 8, 2, 128, 128, BF),
    "blocks of 256": ([900, 131], [60, 2], 8, 2, 128, 256, HF),
    "blocks of 24": ([200, 131], [60, 2], 8, 2, 128, 24, BF),
    "blocks of 1": ([150, 31], [20, 2], 4, 2, 64, 1, BF),
    "head of 96": ([150, 31], [20, 2], 4, 2, 96, 16, BF),
    "head of 20": ([150, 31], [20, 2], 4, 2, 20, 16, HF),
    "fp32": ([150, 31], [20, 2], 4, 2, 128, 16, FP),
}


@pytest.mark.parametrize("name", SHAPES)
def test_chunk_attention_matches_64_bits(name):
    dev = need_gpu()
    case = Case(*SHAPES[name], seed=len(name))
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("name", [n for n in SHAPES if SHAPES[n][4] in (64, 96, 128)])
def test_chunk_attention_over_the_8_bit_cache_matches_64_bits(name):
    dev = need_gpu()
    case = Case(*SHAPES[name], seed=len(name), quant=True)
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("name", ["drafted", "chunk", "mixed with idle and empty sessions", "d 64"])
def test_cuda_core_path(name, quant):
    dev = need_gpu()
    case = Case(*SHAPES[name], seed=3, quant=quant)
    case.check(case.run(dev, path="simt"))
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
def test_many_sessions_and_long_ragged_ones(quant):
    """More sessions than a warp scans at once, more work units than CTAs, and sessions long enough
    to be split over several of them."""
    dev = need_gpu()
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(1, 300, (70,), generator=g).tolist() + [9000, 4097]
    new = [min(s, int(n)) for s, n in zip(lens, torch.randint(0, 5, (72,), generator=g))]
    new[-1] = 70
    case = Case(lens, new, 8, 2, 128, 16, BF, seed=4, quant=quant)
    case.check(case.run(dev))
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("gain", [0.0, 6.0])
def test_flat_and_peaked_logits(gain, quant):
    """All logits equal, and logits tens of units apart (running maxima that rise along the way)."""
    dev = need_gpu()
    case = Case([1000, 300], [130, 1], 8, 2, 128, 16, BF, seed=5, gain=gain, quant=quant)
    order = torch.argsort(case.k[0][:, 0, 0].float())          # rising logits for many queries
    at = C.slots(case.table, 0, 0, 1000, 16)
    case.cache[:, at] = case.cache[:, at[order]]
    case.check(case.run(dev))
    assert_device_clean(dev)


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("path", ["auto", "simt"])
def test_hidden_tokens_do_not_reach_a_query(path, quant):
    """inf and NaN keys and values in later tokens of the chunk: every query that does not see them
    has the same result as without them; the ones that see a NaN value have NaN in that dim."""
    dev = need_gpu()
    case = Case([400], [200], 8, 2, 128, 16, BF, seed=6, quant=quant)
    clean = case.run(dev, path=path)
    at = int(C.slots(case.table, 0, 350, 351, 16))               # query 150 is the first that sees it
    if quant:
        case.cache[:, at, 2 * 128:2 * 128 + 8] = 255
    else:
        case.cache[0, at, :, 5] = math.nan
        case.cache[1, at, :, 7] = math.inf
        case.cache[1, at, :, 8] = math.nan
    dirty = case.run(dev, path=path)
    assert _equal([x[:150] for x in clean], [x[:150] for x in dirty])
    assert torch.isnan(dirty[0][150:]).all() and torch.isnan(dirty[1][150:]).all()
    if not quant:
        case.cache[0, at] = case.k[0][350]
        dirty = case.run(dev, path=path)
        assert _equal([x[:150] for x in clean], [x[:150] for x in dirty])
        assert torch.equal(clean[1], dirty[1])
        assert (dirty[0][150:, :, 7] == math.inf).all() and torch.isnan(dirty[0][150:, :, 8]).all()
        rest = [d for d in range(128) if d not in (7, 8)]
        assert torch.equal(clean[0][:, :, rest], dirty[0][:, :, rest])
    assert_device_clean(dev)


def test_strided_inputs_and_given_outputs():
    """Queries inside a fused projection, one layer of a stacked cache, outputs inside larger ones,
    a scale of the caller's, and a workspace kept between calls of different sizes."""
    dev = need_gpu()
    from actkv_open_b200.kernels.chunk_attn import chunk_workspace
    ws = chunk_workspace(dev)
    for lens, new, seed in (([700, 40], [260, 3], 1), ([90], [1], 2), ([700, 40], [260, 3], 3)):
        case = Case(lens, new, 8, 2, 128, 16, BF, seed=seed)
        t = case.q.shape[0]
        fused = torch.randn(t, 12, 128).to(BF).to(dev)
        fused[:, :8] = case.q.to(dev)
        stack = torch.zeros(3, 2, case.nb, 16, 2, 128, dtype=BF, device=dev)
        stack[1] = case.cache.view(2, case.nb, 16, 2, 128).to(dev)
        table = torch.full((len(lens), case.table.shape[1] + 5), -1, dtype=torch.int32, device=dev)
        table[:, :case.table.shape[1]] = case.table.to(dev)
        out = torch.full((t, 9, 160), 3.0, dtype=BF, device=dev)
        lse = torch.full((t, 10), 3.0, device=dev)
        got = case.run(dev, given=dict(q=fused[:, :8], cache=stack[1], table=table), out=out[:, :8, :128], lse=lse[:, :8],
                       workspace=ws, scale=0.2)
        assert got[0].data_ptr() == out.data_ptr()
        case.check(got, scale=0.2)
        assert (out[:, 8] == 3).all() and (out[:, :, 128:] == 3).all() and (lse[:, 8:] == 3).all()
    assert_device_clean(dev)


def test_layouts_that_tensor_maps_cannot_take():
    """Heads apart from one another, and a cache that starts off a 16-byte boundary: the CUDA cores."""
    dev = need_gpu()
    case = Case([300, 20], [40, 1], 8, 2, 128, 16, BF, seed=8)
    kv = case.device(dev)["cache"]
    apart = torch.zeros(2, case.nb, 2, 16, 128, dtype=BF, device=dev).transpose(2, 3)
    apart.copy_(kv)
    case.check(case.run(dev, given=dict(cache=apart)))
    flat = torch.zeros(kv.numel() + 1, dtype=BF, device=dev)
    odd = flat[1:].view(kv.shape)
    odd.copy_(kv)
    case.check(case.run(dev, given=dict(cache=odd)))
    with pytest.raises(NotImplementedError):
        case.run(dev, given=dict(cache=odd), path="tcgen05")
    assert_device_clean(dev)


@pytest.mark.parametrize("quant", [False, True])
def test_planes_past_32_bit_offsets(quant):
    """Block ids whose element (and byte) offsets pass 2^32, in the V plane and within a plane."""
    dev = need_gpu()
    first = (1 << 32) // (64 * 16 * 8 * 132) * 64 if quant else (1 << 32) // (16 * 8 * 128)
    case = Case([500, 60], [40, 2], 8, 8, 128, 16, BF, seed=10, quant=quant)
    x = case.device(dev)
    big = torch.zeros((2, first + case.nb) + x["cache"].shape[2:], dtype=x["cache"].dtype, device=dev)
    big[:, first:] = x["cache"]
    case.check(case.run(dev, given=dict(cache=big, table=x["table"] + first)))
    assert_device_clean(dev)


def test_other_streams_and_repeats_are_bitwise_equal():
    dev = need_gpu()
    case = Case([3000, 500, 40], [1, 300, 5], 32, 8, 128, 16, BF, seed=11)
    x = case.device(dev)
    want = case.run(dev, given=x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [case.run(dev, given=x) for _ in range(3)]
    side.synchronize()
    assert all(_equal(want, g) for g in got)
    graph = torch.cuda.CUDAGraph()
    from actkv_open_b200.kernels.chunk_attn import chunk_workspace
    ws = chunk_workspace(dev)
    out, lse = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    with torch.cuda.graph(graph):
        case.run(dev, given=x, out=out, lse=lse, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert _equal(want, (out, lse))
    assert_device_clean(dev)


def test_a_one_token_chunk_agrees_with_decode_attention():
    dev = need_gpu()
    from actkv_open_b200.kernels.lse_attn import paged_decode_attention
    case = Case([900, 70, 128], [1, 1, 1], 32, 8, 128, 16, BF, seed=12)
    x = case.device(dev)
    out, lse = case.run(dev, given=x)
    d_out, d_lse = paged_decode_attention(x["q"], x["cache"], x["table"], x["seq"])
    _, _, mag, size = case.ref()
    assert ((out.double() - d_out.double()).abs().cpu() <= (2 * U[BF] + 3e-4) * mag).all()
    assert ((lse - d_lse).abs().cpu().double() <= 4e-5 + 16e-6 * size).all()
    assert_device_clean(dev)


def test_refusals():
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    from actkv_open_b200.kernels.chunk_attn import chunk_workspace
    case = Case([50], [3], 8, 2, 128, 16, BF)
    x = case.device(dev)
    with pytest.raises(RuntimeError, match="CUDA"):
        case.run(dev, given=dict(q=case.q))
    with pytest.raises(AssertionError):
        case.run(dev, given=dict(cache=x["cache"].half()))
    with pytest.raises(AssertionError):
        case.run(dev, given=dict(q=x["q"][:, :7]))
    with pytest.raises(AssertionError):
        case.run(dev, given=dict(q_off=x["q_off"].long()))
    with pytest.raises(AssertionError):
        case.run(dev, given=dict(q_off=x["q_off"][:1]))
    with pytest.raises(AssertionError):
        case.run(dev, out=torch.empty(3, 8, 128, device=dev))
    with pytest.raises(AssertionError, match="scale"):
        case.run(dev, scale=-1.0)
    with pytest.raises(KeyError):
        case.run(dev, path="pair")
    with pytest.raises(RuntimeError, match="workspace"):
        case.run(dev, workspace=chunk_workspace(dev)[:100], path="tcgen05")
    short = torch.zeros(2, case.nb, 16, 200, dtype=torch.uint8, device=dev)
    with pytest.raises(AssertionError, match="short"):
        q8 = Case([50], [3], 8, 2, 128, 16, BF, quant=True)
        q8.run(dev, given=dict(cache=short))
    wide = Case([30], [2], 2, 1, 288, 16, BF)
    with pytest.raises(NotImplementedError, match="256"):
        wide.run(dev)
    # nothing to do: no launch, and outputs of no rows
    none = case.run(dev, given=dict(q=x["q"][:0], q_off=torch.zeros(2, dtype=torch.int32, device=dev)))
    assert none[0].shape == (0, 8, 128)
    assert_device_clean(dev)
    # block ids outside the cache are flagged, not followed
    for bad in (-1, case.nb, 1 << 30):
        for path in ("auto", "simt"):
            case.run(dev, given=dict(table=torch.full_like(x["table"], bad)), path=path)
            torch.cuda.synchronize()
            assert N.read_device_status(dev) == N.DEV_BAD_INDEX
    # a table narrower than the session
    long = Case([50], [3], 8, 2, 128, 16, BF)
    for path in ("auto", "simt"):
        long.run(dev, given=dict(table=x["table"][:, :1], seq=torch.tensor([5000], dtype=torch.int32, device=dev)), path=path)
        torch.cuda.synchronize()
        assert N.read_device_status(dev) == N.DEV_BAD_INDEX
