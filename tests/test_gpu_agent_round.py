"""The pieces together: the host cache's chunk_attention, QuantPagedCache through append, release,
scoring and eviction, and the agent-round example on both caches."""
import os
import sys

import pytest
import torch

import chunk_cases as C
from conftest import ROOT
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(ROOT, "examples"))


def _quant_cache(dev, sessions=3, blocks=64, layers=3, hkv=2, d=128, bs=16, tokens=256):
    from actkv_open_b200.engine import QuantPagedCache
    c = QuantPagedCache(blocks, bs, hkv, d, layers, sessions, tokens, device=dev)
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(3)).tolist()
    c.set_state([[] for _ in range(sessions)], [0] * sessions, order)
    return c


def _rows(c, r):
    """[L, 2, S, row] bytes of session r."""
    tables, seq, _ = c.state()
    pos = torch.arange(seq[r])
    slot = torch.tensor(tables[r] or [0])[pos // c.block_size] * c.block_size + pos % c.block_size
    return c.rows.flatten(2, 3).cpu()[:, :, slot, :c.n_kv_heads * (c.head_dim + c.head_dim // 32)]


def _packed(x, row):
    """[L, n, Hkv, D] -> [L, n, bytes]"""
    n = x.shape[2] * (x.shape[3] + x.shape[3] // 32)
    return torch.stack([C.pack_rows(x[la], row)[:, :n] for la in range(x.shape[0])])


def test_append_quantises_and_allocates_like_the_16_bit_cache():
    dev = need_gpu()
    from actkv_open_b200.engine import DevicePagedCache
    from actkv_open_b200._native import OutOfBlocks
    c = _quant_cache(dev)
    plain = DevicePagedCache(64, 16, 2, 128, 3, 3, 256, device=dev)
    plain.set_state([[]] * 3, [0] * 3, torch.randperm(64, generator=torch.Generator().manual_seed(3)).tolist())
    g = torch.Generator().manual_seed(4)
    kept = [[], [], []]
    for n_new in ([40, 0, 17], [1, 33, 100], [90, 5, 16]):
        k, v = (torch.randn(3, sum(n_new), 2, 128, generator=g).bfloat16() for _ in range(2))
        c.append(k.to(dev), v.to(dev), n_new)
        plain.append(k.to(dev), v.to(dev), n_new)
        at = 0
        for r, n in enumerate(n_new):
            kept[r].append((k[:, at:at + n], v[:, at:at + n]))
            at += n
    assert c.state() == plain.state()
    for r in range(3):
        got = _rows(c, r)
        for p in range(2):
            want = _packed(torch.cat([x[p] for x in kept[r]], 1), c.row_bytes)
            assert torch.equal(got[:, p], want)
    # the first session that does not fit and those after it are left alone, rows and all
    before, state = c.rows.clone(), c.state()
    k = torch.randn(3, 16 + 2000 + 16, 2, 128, generator=g).bfloat16().to(dev)
    with pytest.raises(OutOfBlocks):
        c.append(k, k, [16, 2000, 16])
    tables, seq, _ = c.state()
    assert seq == [state[1][0] + 16, state[1][1], state[1][2]] and tables[1:] == state[0][1:]
    changed = (c.rows != before).any(-1).any(0).any(0).nonzero().tolist()
    assert {b for b, _ in changed} <= set(tables[0]) and len(changed) == 16
    c.release([1])
    assert c.state()[1][1] == 0
    assert_device_clean(dev)


def test_eviction_moves_rows_and_scores_from_the_read_back_keys():
    """A pipeline step over the 8-bit cache does what the same step does over a 16-bit cache that
    holds the read-back rows: scores, kept tokens, tables and (packed again) every kept row."""
    dev = need_gpu()
    from actkv_open_b200.engine import DevicePagedCache, EvictionPipeline
    c = _quant_cache(dev, tokens=256)
    g = torch.Generator().manual_seed(5)
    n_new = [200, 120, 16]
    k, v = (torch.randn(3, sum(n_new), 2, 128, generator=g).bfloat16() for _ in range(2))
    c.append(k.to(dev), v.to(dev), n_new)
    plain = DevicePagedCache(64, 16, 2, 128, 3, 3, 256, device=dev)
    plain.set_state([[]] * 3, [0] * 3, torch.randperm(64, generator=torch.Generator().manual_seed(3)).tolist())
    plain.append(C.quantise_ref(k)[0].bfloat16().to(dev), C.quantise_ref(v)[0].bfloat16().to(dev), n_new)
    q = torch.randn(3, 8 + 8 + 4, 8, 128, generator=g).bfloat16().to(dev)
    done = []
    for cache in (c, plain):
        pipe = EvictionPipeline(cache)
        pipe.set_round([8, 8, 4], [50, 50, 10])
        assert torch.equal(cache.keys16(0, 3)[:, 0, cache.block_table[0, :4].long()],
                           plain.kv[:, 0, plain.block_table[0, :4].long()])
        lse = pipe.region_lse(q).clone()
        pipe.step(q, lse)
        done.append((lse, pipe.heads.clone(), cache.state(), pipe.keep_scores.clone()))
    for a, b in zip(done[0], done[1]):
        assert torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b
    assert done[0][2][1] == [50, 50, 10]
    tables, seq, _ = plain.state()
    for r in range(3):
        pos = torch.arange(seq[r])
        slot = torch.tensor(tables[r])[pos // 16] * 16 + pos % 16
        kept = plain.kv.flatten(2, 3).cpu()[:, :, slot]
        got = _rows(c, r)
        for p in range(2):
            vals = torch.stack([C.unpack_rows(got[la, p], 2, 128) for la in range(3)])
            assert torch.equal(vals, kept[:, p].double())
    # host queries: the grouped launches
    pipe = EvictionPipeline(c)
    pipe.set_round([4, 4, 4], [20, 20, 8])
    qh = torch.randn(3, 12, 8, 128, generator=g).bfloat16()
    lse = pipe.region_lse(qh.to(dev)).cpu()
    pipe.step_host(qh.pin_memory(), lse.pin_memory())
    assert c.state()[1] == [20, 20, 8]
    assert_device_clean(dev)


def test_host_cache_chunk_attention():
    dev = need_gpu()
    from actkv_open_b200.paged import PagedKVCache
    g = torch.Generator().manual_seed(6)
    c = PagedKVCache(40, 16, 2, 128, n_layers=2, dtype=torch.bfloat16, device=dev)
    data = {}
    for r, n in ((0, 90), (1, 33)):
        k, v = (torch.randn(2, n, 2, 128, generator=g).bfloat16() for _ in range(2))
        c.append(r, k.to(dev), v.to(dev))
        data[r] = (k, v)
    q = torch.randn(20 + 33, 8, 128, generator=g).bfloat16()
    out, lse = c.chunk_attention([0, 1], q.to(dev), [20, 33], layer=1)
    want, want_l, mag, size = C.attention_ref(q, C.offsets([20, 33]), lambda r: data[r][0][1], lambda r: data[r][1][1],
                                              [90, 33], 128 ** -0.5)
    assert ((out.cpu().double() - want).abs() <= (2 * 2.0 ** -8 + 1e-4) * mag).all()
    assert ((lse.cpu().double() - want_l).abs() <= 2e-5 + 8e-6 * size).all()
    assert_device_clean(dev)


def test_the_example_on_both_caches():
    """Same lengths on both; the lse of the first round's action tokens, where the two hold the same
    tokens, agrees as far as 8 bits allow: a logit is a sum of 128 products of keys that err by up
    to 1/16 of themselves (rms 1/27), so by about rms |q| |k| 128^0.5 / 27 / 128^0.5 = 1/27 in the
    mean square, and an lse over hundreds of tokens by less."""
    dev = need_gpu()
    import agent_round
    kw = dict(sessions=2, layers=2, hq=8, hkv=2, observe=96, act=16, rounds=3, budget=0.5)
    plain, again, quant = agent_round.run(**kw), agent_round.run(**kw), agent_round.run(quant=True, **kw)
    for (x, lse, lens), (x2, lse2, lens2), (_, lse8, lens8) in zip(plain, again, quant):
        assert torch.equal(x, x2) and torch.equal(lse, lse2)
        assert lens == lens2 == lens8
        assert torch.isfinite(x).all() and torch.isfinite(lse8).all()
    assert (plain[0][1][0] - quant[0][1][0]).abs().max() < 4 / 27
    assert plain[-1][2][0] < 3 * 112
    assert_device_clean(dev)
