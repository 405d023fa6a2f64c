"""Chunk attention where its schedule, its tables and its values leave the ordinary: units that see
nothing among units that do, both tensor-core kernels in one call, sessions of a few rows in every type
and head size, table entries and offsets out of range, values that are not finite.  Bounds as derived in
test_gpu_chunk.py."""
import pytest
import torch

from gpu_util import assert_device_clean, need_gpu
from test_gpu_chunk import BF, Case, U, _equal

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
