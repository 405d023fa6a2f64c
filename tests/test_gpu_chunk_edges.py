"""Chunk attention where its schedule, its tables and its values leave the ordinary: units that see
nothing among units that do, both tensor-core kernels in one call, sessions of a few rows in every type
and head size, table entries and offsets out of range, values that are not finite.  Bounds as derived in
test_gpu_chunk.py."""
import pytest

from gpu_util import assert_device_clean, need_gpu
from test_gpu_chunk import BF, Case, _equal

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
