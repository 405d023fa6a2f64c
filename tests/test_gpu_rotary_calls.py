"""Calls of rotate_write and of the 4-bit cache beyond the plain one: other streams, captured graphs, two calls at once,
planes far apart, expanded heads, wide and narrow ones.  What is compared is exact: the same digits."""
import pytest
import torch

import chunk_cases as C
import quant4_cases as Q
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


class _Call:
    def __init__(self, dev, lens, new, hq, hkv, d, bs, layers, dtype, rot, pairs, bits, seed=0):
        from actkv_open_b200.kernels.quant_cache import quant_row_bytes
        from actkv_open_b200.kernels.rotary import rotary_table
        self.lens, self.hkv, self.d, self.bs, self.layers, self.dtype = lens, hkv, d, bs, layers, dtype
        self.pairs, self.bits = pairs, bits
        self.table, self.nb, self.off, self.q, self.k, self.v, self.pos = Q.new_tokens(
            lens, new, hq, hkv, d, bs, layers, dtype, seed=seed, positions=900)
        self.angles = rotary_table(rot, 900, device="cpu")
        self.tail = (hkv, d) if bits is None else (quant_row_bytes(hkv, d, bits),)
        self.kind = dtype if bits is None else torch.uint8
        self.x = [t.to(dev) for t in (self.q, self.k, self.v, self.pos, self.angles, self.off)]
        self.tables = [self.table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)]
        self.dev = dev

    def cache(self, nb=None):
        return torch.zeros(self.layers, 2, nb or self.nb, self.bs, *self.tail, dtype=self.kind, device=self.dev)

    def run(self, cache, table=None, **kw):
        from actkv_open_b200.kernels.rotary import rotate_write
        return rotate_write(*self.x, cache, self.tables[0] if table is None else table, self.tables[1],
                            interleaved=self.pairs, bits=self.bits, **kw)

    def want(self):
        """(queries, cache) of the formula in 32 bits."""
        cache = torch.zeros(self.layers, 2, self.nb * self.bs, *self.tail, dtype=self.kind)
        tok, slot = Q.written(self.table, self.off, self.lens, self.bs, self.layers)
        k = Q.turn(self.k.float(), self.pos, self.angles, self.pairs)
        for la in range(self.layers):
            for p, x in enumerate((k, self.v.float())):
                if self.bits is None:
                    cache[la, p, slot] = x[la, tok].to(self.dtype)
                else:
                    n = self.hkv * (self.d * self.bits // 8 + self.d // 32)
                    rows = (Q if self.bits == 4 else C).pack_rows(x[la, tok], self.tail[0])
                    cache[la, p, slot, :n] = rows[:, :n]
        return Q.turn(self.q.float(), self.pos, self.angles, self.pairs).to(self.dtype), cache.view(self.cache().shape)


@pytest.mark.parametrize("bits", [None, 8, 4])
def test_other_streams_and_a_captured_call_replayed_on_new_tokens(bits):
    dev = need_gpu()
    a = _Call(dev, [300, 64, 33], [120, 1, 0], 8, 2, 128, 16, 2, BF, 128, False, bits, seed=1)
    b = _Call(dev, [300, 64, 33], [120, 1, 0], 8, 2, 128, 16, 2, BF, 128, False, bits, seed=2)
    a.run(a.cache())
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    got = {}
    for s, c in ((side, a), (other, b)):                   # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            cache = c.cache()
            got[c] = (c.run(cache), cache)
    side.synchronize()
    other.synchronize()
    for c in (a, b):
        q, cache = c.want()
        assert torch.equal(got[c][0].cpu(), q) and torch.equal(got[c][1].cpu(), cache)
    graph, cache, out = torch.cuda.CUDAGraph(), a.cache(), torch.zeros_like(a.x[0])
    with torch.cuda.graph(graph):
        a.run(cache, q_out=out)
    for mine, new in zip(a.x, b.x):                        # the next tokens, in the captured call's tensors
        mine.copy_(new)
    a.tables[0].copy_(b.tables[0])
    graph.replay()
    torch.cuda.synchronize()
    q, want = b.want()
    assert torch.equal(out.cpu(), q) and torch.equal(cache.cpu(), want)
    assert_device_clean(dev)


@pytest.mark.parametrize("bits", [None, 4])
def test_blocks_and_layers_past_32_bit_offsets(bits):
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read
    c = _Call(dev, [60, 20], [33, 20], 8, 8, 128, 16, 2, BF, 128, False, bits, seed=3)
    row = c.tail[0] if bits else 8 * 128
    first = (1 << 31) // (16 * row) + 64                   # over 2^31 elements before a plane's first block
    cache = c.cache(first + c.nb)
    out = c.run(cache, table=c.tables[0] + first)
    q, want = c.want()
    assert torch.equal(out.cpu(), q) and torch.equal(cache[:, :, first:].cpu(), want)
    assert not cache[:, :, :first].any()
    if bits:
        args = (8, 128, c.x[5])
        far = dequantize_read(cache, *args, c.tables[0] + first, c.tables[1], 53, bits=4)
        near = dequantize_read(cache[:, :, first:].contiguous(), *args, *c.tables, 53, bits=4)
        assert all(torch.equal(x, y) for x, y in zip(far, near))
    assert_device_clean(dev)


@pytest.mark.parametrize("d, rot, dtype", [(512, 512, FP), (512, 64, BF), (544, 32, HF), (8, 8, BF), (24, 8, HF), (256, 40, FP),
                                           (2, 2, BF)])
@pytest.mark.parametrize("pairs", [False, True])
def test_wide_and_narrow_heads(d, rot, dtype, pairs):
    dev = need_gpu()
    c = _Call(dev, [20, 9], [13, 9], 5, 3, d, 4, 2, dtype, rot, pairs, None, seed=d)
    cache = c.cache()
    out = c.run(cache)
    q, want = c.want()
    assert torch.equal(out.cpu(), q) and torch.equal(cache.cpu(), want)
    assert_device_clean(dev)


@pytest.mark.parametrize("d, rot", [(32, 32), (32, 8), (64, 40), (160, 128), (544, 544)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("bits", [8, 4])
def test_rows_of_other_heads(d, rot, pairs, bits):
    dev = need_gpu()
    c = _Call(dev, [20, 9], [13, 9], 5, 3, d, 4, 2, BF, rot, pairs, bits, seed=d)
    cache = c.cache()
    out = c.run(cache)
    q, want = c.want()
    assert torch.equal(out.cpu(), q) and torch.equal(cache.cpu(), want)
    assert_device_clean(dev)


@pytest.mark.parametrize("bits", [None, 8, 4])
def test_expanded_heads_and_tokens(bits):
    dev = need_gpu()
    c = _Call(dev, [70, 33], [40, 33], 4, 4, 64, 16, 2, BF, 64, False, bits, seed=5)
    # one key and value head for all four, the same query for every token
    k, v, q = c.k[:, :, :1], c.v[:, :, :1], c.q[:, :1]
    whole = [x.contiguous() for x in (q.expand_as(c.q), k.expand_as(c.k), v.expand_as(c.v))]
    c.q, c.k, c.v = whole
    c.x[:3] = [q.to(dev).expand_as(c.q), k.to(dev).expand_as(c.k), v.to(dev).expand_as(c.v)]
    cache = c.cache()
    out = c.run(cache)
    want_q, want = c.want()
    assert torch.equal(out.cpu(), want_q) and torch.equal(cache.cpu(), want)
    assert_device_clean(dev)


def test_queries_that_are_not_finite_stay_in_their_pairs():
    dev = need_gpu()
    c = _Call(dev, [20], [20], 2, 2, 64, 16, 1, BF, 64, False, None, seed=6)
    c.q[0, 3, 1, 5], c.k[0, 4, 0, 40] = float("inf"), float("nan")
    c.x[0], c.x[1] = c.q.to(dev), c.k.to(dev)
    cache = c.cache()
    out = c.run(cache).cpu()
    q, want = c.want()
    assert torch.equal(out.nan_to_num(7.0), q.nan_to_num(7.0)) and torch.equal(cache.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert int((~out.isfinite()).sum()) == 2 and int((~cache.isfinite()).sum()) == 2


def test_write_and_read_in_4_bits_captured_and_at_once():
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import dequantize_read, quantize_write
    c = [_Call(dev, [300, 64], [120, 64], 2, 2, 64, 16, 2, HF, 64, False, 4, seed=s) for s in (7, 8)]

    def run(x, rows, k=None, v=None):
        quantize_write(x.x[1], x.x[2], x.x[5], rows, *x.tables, bits=4)
        return dequantize_read(rows, 2, 64, x.x[5], *x.tables, 184, dtype=HF, k_out=k, v_out=v, bits=4)

    want = [run(x, x.cache()) for x in c]
    for x, w in zip(c, want):
        for part, ref in ((w[0], x.k), (w[1], x.v)):
            assert torch.equal(part.cpu(), Q.quantise_ref(ref)[0].clamp(-65504, 65504).to(HF))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in c], []
    for s, x in zip(streams, c):
        with torch.cuda.stream(s):
            got.append(run(x, x.cache()))
    for s in streams:
        s.synchronize()
    rows, k, v = c[0].cache(), torch.zeros_like(want[0][0]), torch.zeros_like(want[0][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(c[0], rows, k, v)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for g, w in zip(got + [(k, v)], want + [want[0]]):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    assert_device_clean(dev)


def test_two_attentions_over_4_bits_at_once():
    dev = need_gpu()
    from test_gpu_chunk import _equal
    from test_gpu_chunk4 import Case4
    cases = [Case4([3001, 500], new, 32, 8, 128, 16, BF, seed=20) for new in ([1, 3], [1, 200])]
    xs = [c.device(dev) for c in cases]
    want = [c.run(dev, given=x) for c, x in zip(cases, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(4):
        for s, c, x in zip(streams, cases, xs):
            with torch.cuda.stream(s):
                got.append(c.run(dev, given=x))
    for s in streams:
        s.synchronize()
    assert all(_equal(want[i % 2], g) for i, g in enumerate(got))
    assert_device_clean(dev)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("d, dtype, pairs", [(128, BF, False), (64, HF, True)])
def test_queries_so_large_that_they_go_apart(d, dtype, pairs, bits):
    dev = need_gpu()
    from actkv_open_b200.kernels.quant_cache import quant_row_bytes
    from actkv_open_b200.kernels.rotary import rotary_table, rotate_write
    n = (1 << 26) // (32 * d) + 77
    gen = torch.Generator(device=dev).manual_seed(d)
    q, k, v = (torch.randn(1, n, h, d, generator=gen, device=dev).to(dtype) for h in (32, 2, 2))
    blocks = -(-n // 16)
    table = torch.randperm(blocks, generator=gen, device=dev).int()[None]
    pos = torch.randint(0, 900, (n + 3,), generator=gen, device=dev, dtype=torch.int32)[:n]
    pos[5] = 900                                           # a position that the angles do not have
    rest = (pos, rotary_table(d, 900), torch.tensor([0, n - 20], dtype=torch.int32, device=dev))
    seq = torch.tensor([n - 20], dtype=torch.int32, device=dev)

    def run(q, cache, bits, out=None):
        return rotate_write(q, k, v, *rest, cache, table, seq, q_out=out, interleaved=pairs, bits=bits)

    from actkv_open_b200 import _native as N
    row = quant_row_bytes(2, d, bits)
    rows, alone = (torch.zeros(1, 2, blocks, 16, row, dtype=torch.uint8, device=dev) for _ in range(2))
    got, want = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
    N.read_device_status(dev)
    run(q, rows, bits, got)
    assert N.read_device_status(dev) == N.DEV_BAD_INDEX
    run(None, alone, bits)
    run(q, torch.zeros(1, 2, blocks, 16, 2, d, dtype=dtype, device=dev), None, want)
    assert torch.equal(rows, alone) and bool(rows.any())
    assert torch.equal(got, want) and bool((got[:, [5] + list(range(n - 20, n))] == 9.0).all())
    N.read_device_status(dev)
