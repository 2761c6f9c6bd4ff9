"""Batches that reach every kernel of the paged attention, named by the items that the plan cuts them into
(tests/test_paged_plan.py holds them to it on the CPU, tests/test_paged_tiles_gpu.py runs them)."""
from pathlib import Path
from typing import NamedTuple

import numpy as np

from tests.paged_ref import Case

ROOT = Path(__file__).resolve().parents[1]


class Batch(NamedTuple):
    n: list        # new tokens of each sequence
    past: list     # own tokens before them
    prefix: int
    kv: int
    group: int
    narrow: tuple  # (rows of a prefix item or 0, rows of an own item) at d_head up to 64 …
    wide: tuple    # … and beyond
    cut: bool      # records and a join (else items write the output themselves)
    page: int = 16

    @property
    def length(self):
        return [x + y for x, y in zip(self.n, self.past)]

    def case(self, dh, dtype, seed=0, **kw):
        return Case(np.random.default_rng(1000 * seed + dh + len(self.n)), self.n, self.length, self.prefix, self.page,
                    self.kv, self.group, dh, dtype, **kw)


def _ragged(b, lo, hi):
    return [lo + (7 * i) % (hi - lo + 1) for i in range(b)]


# A sequence's own axis, prefix and own keys on it: causal masks, the crossing from the prefix's pages (whose
# last one is partly used) to the sequence's, tiles that end behind the last row.
OWN = {
    "64 rows": Batch([40, 33, 60, 64], [40, 0, 7, 300], 2099, 2, 1, (0, 64), (0, 64), True),
    "64 rows, group 4": Batch([10, 0, 16, 3], [40, 5, 0, 130], 2099, 2, 4, (0, 64), (0, 64), True, 32),
    "128 rows": Batch([100, 65, 90], [40, 0, 7], 2150, 2, 1, (0, 128), (0, 128), True),
    "128 rows, group 2": Batch([34, 50, 41], [140, 0, 7], 2150, 2, 2, (0, 128), (0, 128), True, 8),
    "256 rows": Batch([200, 131, 150], [40, 0, 7], 2150, 2, 1, (0, 256), (0, 128), True),
    "several tiles": Batch([300, 2, 259], [0, 90, 33], 2500, 2, 1, (0, 256), (0, 128), True, 64),
    "several tiles, group 3": Batch([100, 61], [1, 500], 2100, 3, 3, (0, 256), (0, 128), True, 4),
    "128 rows of many axes": Batch(_ragged(25, 65, 80), [0, 7, 20, 69, 1] * 5, 100, 16, 1, (0, 128), (0, 128), False),
    "256 rows of many axes": Batch(_ragged(9, 257, 270), [0, 7, 60, 1, 31, 12, 0, 8, 64], 97, 16, 1, (0, 256), (0, 128), False),
    "16 rows of one sequence": Batch([21], [30], 77, 1, 1, (0, 16), (0, 16), False),
    "one row": Batch([1, 1, 0, 1], [40, 0, 9, 500], 130, 2, 1, (0, 16), (0, 16), True),
    "two rows": Batch([1, 1, 0, 1], [40, 0, 9, 500], 130, 2, 2, (0, 16), (0, 16), True),
    "three rows": Batch([1, 1, 0, 1], [40, 0, 9, 500], 130, 2, 3, (0, 16), (0, 16), True),
}
# The prefix read once for all: its items hold the rows of every sequence.
POOLED = {
    "prefix 16, own 1": Batch([1] * 20, _ragged(20, 0, 36), 1300, 3, 1, (16, 16), (16, 16), True),
    "prefix 16, own 2": Batch([1] * 14, _ragged(14, 0, 36), 1900, 3, 2, (16, 16), (16, 16), True),
    "prefix 16, own 4": Batch([1] * 9, _ragged(9, 0, 36), 2500, 4, 3, (16, 16), (16, 16), True),
    "prefix 16, own 16": Batch([3, 2, 3, 1, 3], _ragged(5, 0, 36), 5611, 4, 2, (16, 16), (16, 16), True),
    "prefix 64, own 1": Batch([1] * 40, _ragged(40, 0, 36), 901, 2, 1, (64, 16), (64, 16), True),
    "prefix 64, own 2": Batch([1] * 40, _ragged(40, 0, 36), 901, 2, 2, (64, 16), (64, 16), True),
    "prefix 64, own 4": Batch([1] * 23, _ragged(23, 0, 36), 1700, 2, 4, (64, 16), (64, 16), True),
    "prefix 64, own 16": Batch([3] * 20 + [1], _ragged(21, 0, 36), 1201, 3, 2, (64, 16), (64, 16), True),
    "prefix 64, own 64": Batch([9, 9, 0, 9, 7], _ragged(5, 0, 700), 4201, 8, 3, (64, 64), (64, 64), True),
    "one prompt among steps": Batch([17] + [1] * 9, _ragged(10, 0, 300), 2222, 4, 1, (64, 64), (64, 64), True),
    "prefix 256, own 16": Batch([1] * 90, _ragged(90, 0, 36), 401, 2, 3, (256, 16), (128, 16), True),
    "prefix 256, own 64": Batch([9, 8, 0, 9] * 3, _ragged(12, 0, 200), 2601, 3, 4, (256, 64), (128, 64), True, 128),
}
ALL = {**OWN, **POOLED}
D_HEADS = [8, 24, 32, 40, 64, 80, 128]


def kernels(plan):
    """Names of what a call with this plan launches: (rows of a step's own items, of the prefix's beside
    them) or the rows of a tile kernel's items; and the join."""
    tiles, own = plan["head_tiles"], plan["o_tile"]
    out = set()
    if plan["p_tile"] > 64 or plan["p_tile"] == 64 and own == 64:
        out.add((tiles, "tile", plan["p_tile"]))
    if own > 16:
        out.add((tiles, "tile", own))
    else:
        beside = plan["p_tile"] if plan["p_tile"] <= 64 else 0
        out.add((tiles, "step", plan["step_rows"], 0 if plan["step_rows"] == 16 and beside == 16 else beside))
    return out


def every_kernel(f32):
    out = set()
    for tiles in (1, 2, 3, 4, 6, 8):
        out |= {(tiles, "tile", r) for r in ((64, 128, 256) if tiles <= 4 else (64, 128))}
        for rows in (1, 2, 4, 16) if f32 else (1, 2, 16):
            out |= {(tiles, "step", rows, pre) for pre in ((0, 64) if rows == 16 else (0, 16, 64))}
    return out


def attention_blocks(c, loss=0.0):
    """tests.paged_ref.attention(c), its values and bounds, in products over whole heads of a sequence.  A
    score is a sum of its own, so an infinity or NaN among the keys stays with its key; one among the values
    is taken out of the product and added to the rows that see it.  The bounds are those of the finite rest.

    `loss`: keys, scaled queries and values are exact to so much only, besides their roundings; a score is
    then off by loss·(Σ|q|/√dh + Σ|k|) more, an output by what that makes of its weights and by loss."""
    d, g = c.h * c.dh, c.h // c.kv
    out, lse = np.full((c.n_tok, d), np.nan), np.full((c.n_tok, c.h), np.nan)
    tol, tol_lse = np.zeros((c.n_tok, d)), np.zeros((c.n_tok, c.h))
    for s in range(c.b):
        n = int(c.n[s])
        if n == 0:
            continue
        k, v, there = c.keys(s)
        k, v = np.where(there[:, None, None], k, 0.0), np.where(there[:, None, None], v, 0.0)
        lo = int(c.off[s])
        last = np.maximum(c.prefix + c.length[s] - n + np.arange(n) + 1, c.prefix)
        sees = there[None] & (np.arange(len(k))[None] < last[:, None])
        sees = np.repeat(sees, g, 0)  # rows (token, head of the group)
        count = sees.sum(1)
        for hk in range(c.kv):
            heads = slice(hk * g, (hk + 1) * g)
            q = c.q[lo:lo + n].astype(np.float64).reshape(n, c.h, c.dh)[:, heads].reshape(n * g, c.dh)
            kk, vv = np.ascontiguousarray(k[:, hk]), np.ascontiguousarray(v[:, hk])
            with np.errstate(invalid="ignore"):
                sc = np.where(sees, q @ kk.T / np.sqrt(c.dh), -np.inf)
            size = np.where(sees, np.abs(q) @ np.abs(np.where(np.isfinite(kk), kk, 0.0)).T, 0.0).max(1, initial=0.0)
            delta = (c.dh + 4) * 2.0**-24 * size / np.sqrt(c.dh)
            if loss:
                delta = delta + loss * (np.abs(q).sum(1) / np.sqrt(c.dh) + np.abs(kk).sum(1).max(initial=0.0))
            m = sc.max(1, initial=-np.inf)
            with np.errstate(invalid="ignore"):
                p = np.exp(sc - np.where(np.isneginf(m), 0.0, m)[:, None])
            l = p.sum(1)
            some = ~(l <= 0)  # NaN too
            w = p / np.where(some, l, 1.0)[:, None]
            sums = (4 * np.sqrt(count) + 24) * 2.0**-24
            put = lambda dst, x: dst[lo:lo + n].reshape(n, c.kv, -1)[:, hk].__setitem__(  # noqa: E731
                slice(None), x.reshape(n, -1))
            vf = np.where(np.isfinite(vv), vv, 0.0)
            o = w @ vf
            for key, col in np.argwhere(~np.isfinite(vv)):
                o[sees[:, key], col] += w[sees[:, key], key] * vv[key, col]
            put(out, o)
            put(tol, ((2 * delta + sums)[:, None] * (w @ np.abs(vf)) + loss))
            ll = np.where(some, np.where(some, m, 0.0) + np.log(np.where(some, l, 1.0)), -np.inf)
            put(lse, ll)
            put(tol_lse, np.where(some, delta + sums + 2.0**-22 * np.abs(np.where(some, ll, 0.0)), 0.0))
    return out, lse, tol, tol_lse
