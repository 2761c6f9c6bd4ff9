"""The 8-bit cache's attention at the ends of its items' arithmetic, on the GPU, against float64."""
import numpy as np
import pytest

from tests.e4m3_ref import Case8
from tests.test_e4m3_gpu import Device8
from tests.test_paged_gpu import _check

pytestmark = pytest.mark.gpu

# New tokens, prefix, group: single tokens by vector instructions, rows in registers, prefix items of 16, 64 and more
# rows that are joined, tiles of many rows.
ITEMS = [([1, 1, 1], 400, 1), ([1, 1], 6000, 4), ([1] * 40, 3000, 1), ([1] * 90, 500, 3), ([5, 6], 30, 1), ([3] * 3, 2500, 2),
         ([90, 70], 60, 1), ([90, 70], 3000, 1), ([300], 900, 2)]


@pytest.mark.parametrize("n,prefix,group", ITEMS)
@pytest.mark.parametrize("v_e", [94, 100, 104, 112])
@pytest.mark.parametrize("equal", [False, True])
def test_values_near_the_largest(ctx, n, prefix, group, v_e, equal):
    """V of up to 2^115, whose sums over up to 6020 keys stay below 2^128 with weights of at most 1: also where all
    keys weigh the same and every range's sum adds to the others'."""
    c = Case8(np.random.default_rng(v_e + len(n)), n, [x + 20 for x in n], prefix, 16, 1, group, 64, 8)
    c.vs = np.where(c.vs == 255, 255, c.vs.astype(int) + v_e).astype(np.uint8)
    if equal:
        c.q[:] = 0
        c.vb &= 127  # no sign
    with np.errstate(invalid="ignore"):
        c.refresh()
    dev = Device8(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


@pytest.mark.parametrize("n,prefix,group", ITEMS)
@pytest.mark.parametrize("k_e,v_e", [(0, -100), (0, -70), (-100, 0), (-70, 0), (-90, -90), (60, 60)])
def test_the_size_of_all_scales_changes_no_bit(ctx, n, prefix, group, k_e, v_e):
    """Scales of one power of two more, for which the queries make up: the same products, so the same bits times that
    power, whatever stands in a last tile's places without a key."""
    c = Case8(np.random.default_rng(4), n, [x + 23 for x in n], prefix, 16, 1, group, 64, 8)
    got = []
    for k, v in ((0, 0), (k_e, v_e)):
        c.ks = np.where(c.ks == 255, 255, c.ks.astype(int) + k).astype(np.uint8)
        c.vs = np.where(c.vs == 255, 255, c.vs.astype(int) + v).astype(np.uint8)
        c.q *= np.float32(2.0**-k)
        dev = Device8(ctx, c)
        dev.attend()
        got.append(dev.result())
        dev.free()
    rows = int(c.off[-1])
    assert np.array_equal(got[1][0][:rows], got[0][0][:rows] * np.float32(2.0**v_e))
    assert np.array_equal(got[1][1], got[0][1])
