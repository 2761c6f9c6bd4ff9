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


def _queries(dh):
    """Pairs (c, d) of float32 queries whose products with the kernels' float32 factor log2(e)/sqrt(dh) are
    x = (A + 1)·2^5 - 2^-8, 13 ones at the end of its 24 bits, and (A + 1)·2^5, 2^10 <= A < 2^11: with two 11-bit parts
    cut toward zero x loses 3·2^-8, with parts to nearest nothing."""
    factor = (np.float32(1) / np.sqrt(np.float32(dh))) * np.float32(1.44269504088896340736)
    found = []
    for a in range(1024, 2046):
        pair = []
        for x in ((a + 1) * 32 - 2.0**-8, (a + 1) * 32.0):
            near = np.float32(x / float(factor))
            near = [np.nextafter(near, np.float32(s * 1e9)) for s in (-1, 1)] + [near]
            pair.append(next((c for c in near if float(c * factor) == x), None))
        # the roundings of the two products do not stand in for the loss that is looked for
        if None not in pair:
            off = [float(c) * float(factor) - x for c, x in zip(pair, ((a + 1) * 32 - 2.0**-8, (a + 1) * 32.0))]
            if off[0] - off[1] >= 0:
                found.append(pair)
    return np.array(found, np.float32)


@pytest.mark.parametrize("n,prefix,group", [x for x in ITEMS if x[0] != [1, 1, 1]])
@pytest.mark.parametrize("dh", [8, 40, 64, 128])
def test_queries_keep_their_last_bits(ctx, n, prefix, group, dh):
    """Scores (c - d)/√dh of columns that nearly cancel.  x and d's product are rounded once each, 2^-9 at most, the
    sum of the two products once more, 2^-9, in log2: with 2^-10 for all that is smaller 3.5·2^-9; parts that are cut
    lose 6·2^-9."""
    c = Case8(np.random.default_rng(5), n, [x + 23 for x in n], prefix, 16, 1, group, dh, 8)
    c.kb[:] = 0
    c.kb[:, 0], c.kb[:, 1], c.ks[:] = 0x38, 0xb8, 127  # 1 and -1
    c.refresh()
    pairs = _queries(dh)
    assert len(pairs) > 1
    rows = np.arange(c.q.shape[0] * c.h) % len(pairs)
    q = np.zeros((c.q.shape[0] * c.h, dh), np.float32)
    q[:, :2] = pairs[rows]
    c.q = q.reshape(c.q.shape)
    dev = Device8(ctx, c)
    dev.attend()
    out, lse = dev.result()
    dev.free()
    t = np.arange(int(c.off[-1]))
    s = np.searchsorted(c.off[1:], t, side="right")
    keys = c.prefix + np.asarray(c.length)[s] - np.asarray(c.n)[s] + t - np.asarray(c.off)[s] + 1
    exact = (pairs[:, 0].astype(np.float64) - pairs[:, 1]) / np.sqrt(dh)
    want = exact[rows].reshape(-1, c.h)[: len(t)] + np.log(keys)[:, None]
    err = np.abs(lse[: len(t)] - want)
    print(f"{err.max() / (2.0**-9 * np.log(2)):.2f} of 3.5")
    assert err.max() <= 3.5 * 2.0**-9 * np.log(2)


@pytest.mark.parametrize("n,prefix,group", ITEMS)
def test_items_whose_first_keys_are_not_there(ctx, n, prefix, group):
    """Pages that are not there at the start of both axes, so that whole tiles and items have no key."""
    c = Case8(np.random.default_rng(6), n, [x + 150 for x in n], prefix, 16, 1, group, 64, 8)
    c.prefix_pages[: len(c.prefix_pages) // 2] = -1
    c.pages[:, :8] = c.n_pages + 3
    dev = Device8(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()
