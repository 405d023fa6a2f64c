"""Room set aside for new tokens where it does not suffice: nothing is written over the tokens of the sessions that were
refused, with the status read in between or not, and in a captured step."""
import pytest
import torch

import quant4_cases as Q
from gpu_util import assert_device_clean, need_gpu

pytestmark = pytest.mark.gpu


def _cache(dev, bits, blocks, sessions=3, layers=2, hkv=2, d=128, tokens=256):
    from actkv_open_b200.engine import DevicePagedCache, QuantPagedCache
    c = DevicePagedCache(blocks, 16, hkv, d, layers, sessions, tokens, device=dev) if bits == 16 else \
        QuantPagedCache(blocks, 16, hkv, d, layers, sessions, tokens, device=dev, bits=bits)
    c.set_state([[] for _ in range(sessions)], [0] * sessions, list(range(blocks)))
    return c


def _bytes(c, r, first, last):
    """The rows of tokens [first, last) of session r as bytes, every layer and plane."""
    tables, _, _ = c.state()
    pos = torch.arange(first, last)
    slot = (torch.tensor(tables[r])[pos // 16] * 16 + pos % 16).to(c.kv.device)
    return c.kv.flatten(2, 3)[:, :, slot].contiguous().view(torch.uint8).cpu()


def _inputs(dev, n_new, seed, layers=2, hkv=2, d=128):
    g = torch.Generator().manual_seed(seed)
    n = sum(n_new)
    k, v = (torch.randn(layers, n, hkv, d, generator=g).bfloat16().to(dev) for _ in range(2))
    q = torch.randn(layers, n, 4, d, generator=g).bfloat16().to(dev)
    return q, k, v, torch.randint(0, 400, (n,), generator=g).int().to(dev)


@pytest.mark.parametrize("check", [False, True])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_sessions_without_room_keep_their_tokens(bits, check):
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    from actkv_open_b200.kernels.rotary import rotary_table
    angles = rotary_table(128, 400, device=dev)
    c, other = _cache(dev, bits, 8), _cache(dev, bits, 8)
    start = [20, 30, 40]                         # 2, 2 and 3 blocks: one is left
    _, k, v, _ = _inputs(dev, start, 1)
    for x in (c, other):
        x.append(k, v, start)
    new = [14, 20, 3]                            # session 0 takes it, session 1 has none, session 2's fit where they are
    q, k, v, pos = _inputs(dev, new, 2)
    old = [_bytes(c, r, 0, start[r]) for r in range(3)]
    if check:
        with pytest.raises(N.OutOfBlocks) as e:
            c.reserve(new)
        off = e.value.off
        assert e.value.fits == [True, False, False]
    else:
        off = c.reserve(new, check=False)
    assert off.tolist() == [0, 14, 34, 37] and c.state()[1] == [34, 30, 40]
    turned = [c.write_rotated(la, q[la], k[la], v[la], pos, angles, off) for la in range(2)]
    torch.cuda.synchronize()
    assert N.read_device_status(dev) == (0 if check else N.DEV_OUT_OF_BLOCKS)
    assert torch.equal(torch.stack(turned).cpu(), Q.turn(q.float().cpu(), pos.cpu(), angles.cpu(), False).bfloat16())
    assert all(torch.equal(_bytes(c, r, 0, start[r]), old[r]) for r in range(3))
    # the session that fitted has what it has without the others
    alone = other.reserve([14, 0, 0])
    for la in range(2):
        other.write_rotated(la, None, k[la, :14], v[la, :14], pos[:14], angles, alone)
    assert other.state()[1] == [34, 30, 40] and torch.equal(_bytes(c, 0, 0, 34), _bytes(other, 0, 0, 34))
    # room for the others once session 0 is gone; the flags are the last reserve's
    for x in (c, other):
        x.release([0])
        off = x.reserve([0, 20, 3])
        for la in range(2):
            x.write_rotated(la, None, k[la, 14:], v[la, 14:], pos[14:], angles, off)
    assert c.state()[1] == [0, 50, 43]
    for r, s in ((1, 50), (2, 43)):
        assert torch.equal(_bytes(c, r, 0, start[r]), old[r])
        assert torch.equal(_bytes(c, r, start[r], s), _bytes(other, r, start[r], s))
    assert_device_clean(dev)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_a_captured_step_that_runs_out_of_blocks(bits):
    dev = need_gpu()
    from actkv_open_b200 import _native as N
    from actkv_open_b200.kernels.rotary import rotary_table
    angles = rotary_table(128, 400, device=dev)
    c = _cache(dev, bits, 7)
    _, k, v, _ = _inputs(dev, [30, 29, 28], 3)   # 2 blocks each: one is left
    c.append(k, v, [30, 29, 28])
    off = torch.arange(4, dtype=torch.int32, device=dev)
    q, k, v, pos = _inputs(dev, [1, 1, 1], 4)

    def step():
        c.reserve(off, check=False)
        return c.write_rotated(0, q[0], k[0], v[0], pos, angles, off)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = c.state()[1]
    assert seen == [31, 30, 29]
    graph.replay()                               # 32, 31, 30
    graph.replay()                               # 33 (the last block), 32, 31
    assert c.state()[1] == [33, 32, 31] and N.read_device_status(dev) == 0
    old = [_bytes(c, r, 0, s) for r, s in enumerate((33, 32, 31))]
    k.add_(1)
    for n in range(3):
        out.zero_()
        graph.replay()                           # session 1 needs a block: it and session 2 stay
        torch.cuda.synchronize()
        assert N.read_device_status(dev) == N.DEV_OUT_OF_BLOCKS
        assert c.state()[1] == [34 + n, 32, 31]
        assert torch.equal(_bytes(c, 0, 0, 33), old[0])
        assert all(torch.equal(_bytes(c, r, 0, len(old[r][0, 0])), old[r]) for r in (1, 2))
        assert torch.equal(out.cpu(), Q.turn(q[:1].float().cpu(), pos.cpu(), angles.cpu(), False)[0].bfloat16())
    del graph


def test_flags_of_what_fits_are_checked():
    dev = need_gpu()
    from actkv_open_b200.kernels.rotary import rotary_table, rotate_write
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)                                      # noqa: E731
    q, k, v, pos = _inputs(dev, [2, 1], 5)
    angles = rotary_table(128, 400, device=dev)
    cache = torch.zeros(2, 2, 2, 16, 2, 128, dtype=torch.bfloat16, device=dev)
    call = lambda fits: rotate_write(q, k, v, pos, angles, i32(0, 2, 3), cache, i32(0, 1).view(2, 1), i32(5, 1), fits=fits)  # noqa: E731
    out = call(i32(0, 1))
    assert torch.equal(out, call(None)) and (cache[:, :, 0, 3:5] != 0).any()
    cache.zero_()
    call(i32(0, 7))
    assert (cache[:, :, 0] == 0).all() and torch.equal(cache[:, 1, 1, 0], v[:, 2])
    for bad in (i32(1), i32(1, 1).long(), i32(1, 1, 1)[::2][:1]):
        with pytest.raises(AssertionError, match="fits"):
            call(bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(torch.ones(2, dtype=torch.int32))
    assert_device_clean(dev)
