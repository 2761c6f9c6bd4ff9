"""The paged K/V cache in 8 bits and the choice of the next token, from their definitions, with numpy alone.

A pool holds e4m3 numbers (sign, 4 bits of exponent, 3 of significand, 127 a NaN) as bytes, and for every
`block` tokens of a head the byte e + 127 of a power of two 2^e that multiplies them."""
from fractions import Fraction

import numpy as np

from tests.paged_ref import Case

LEAST, MOST = -117, 119  # exponents that an append gives


def _number(byte):
    e, m = (byte >> 3) & 15, byte & 7
    x = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0**-9)
    return np.where(byte & 127 == 127, np.nan, np.where(byte & 128, -x, x))


NUMBERS = _number(np.arange(256))  # float64
_SIZES = NUMBERS[:127]             # ascending


def nearest(x):
    """Bytes of the nearest numbers to x (float64), ties to the even byte; NaN and infinities to NaN."""
    size = np.minimum(np.abs(x), 448.0)
    up = np.clip(np.searchsorted(_SIZES, size), 1, 126)  # exact: numbers and halves of their steps are float64
    low, high = _SIZES[up - 1], _SIZES[up]
    take = np.where(size - low < high - size, up - 1, np.where(size - low > high - size, up, up - up % 2))
    take = np.where(size == 0, 0, take)
    return np.where(np.isfinite(x), take | np.where(np.signbit(x), 128, 0), 127).astype(np.uint8)


def least_exponent(values):
    """The least e with |x| <= 448·2^e for all finite values."""
    v = np.abs(values[np.isfinite(values)]).astype(np.float64)
    top = float(v.max(initial=0.0))
    e = LEAST
    while e < MOST and top > 448.0 * 2.0**e:
        e += 1
    return e


def value(byte, scale):
    with np.errstate(over="ignore"):
        return NUMBERS[byte] * 2.0 ** (np.asarray(scale, np.float64) - 127.0)


class Case8(Case):
    """A Case whose pools hold bytes kb, vb [rows, kv*dh] and scales ks, vs [n_pages, kv, page/block]; kp and vp
    are the values that they stand for.  Unused rows hold NaN, scales of unused blocks 255."""

    def __init__(self, rng, n, length, prefix=0, page=16, kv=2, group=1, dh=32, block=None, sizes=None, **kw):
        super().__init__(rng, n, length, prefix, page, kv, group, dh, "f32", **kw)
        self.dtype, self.block = "e4m3", block or page
        self.kb, self.ks = self._held(self.kp, rng, sizes)
        self.vb, self.vs = self._held(self.vp, rng, sizes)
        self.refresh()

    def _held(self, pool, rng, sizes):
        nb = self.page // self.block
        x = pool.reshape(self.n_pages, nb, self.block, self.kv, self.dh).astype(np.float64)
        if sizes:  # blocks of different magnitudes
            x *= 2.0 ** rng.integers(sizes[0], sizes[1] + 1, (self.n_pages, nb, 1, self.kv, 1))
        top = np.nanmax(np.where(np.isnan(x), 0.0, np.abs(x)), axis=(2, 4))
        e = np.clip(np.ceil(np.log2(np.maximum(top, 1e-300) / 448.0)), LEAST, MOST)
        used = ~np.isnan(x).all(axis=(2, 4))
        byte = nearest(x * 2.0 ** -e[:, :, None, :, None])
        scale = np.where(used, e + 127, 255).astype(np.uint8).transpose(0, 2, 1)
        return byte.reshape(-1, self.kv * self.dh), np.ascontiguousarray(scale)

    def refresh(self):
        """kp and vp from the bytes."""
        for name, byte, scale in (("kp", self.kb, self.ks), ("vp", self.vb, self.vs)):
            s = np.repeat(scale.transpose(0, 2, 1), self.block, 1).reshape(-1, self.kv)
            x = value(byte.reshape(-1, self.kv, self.dh), s[:, :, None])
            setattr(self, name, x.reshape(len(byte), -1).astype(np.float32))

    def append(self, k, v):
        """Rows k, v [n_tok, kv, dh] (float32, k rotated) of the new tokens into the bytes."""
        S = self.block
        for byte, scale, x in ((self.kb, self.ks, k), (self.vb, self.vs, v)):
            byte = byte.reshape(-1, self.kv, self.dh)
            for s in range(self.b):
                past = int(self.length[s] - self.n[s])
                j = max(past, 0)
                while j < self.length[s]:
                    lo, hi = j // S * S, min(j // S * S + S, int(self.length[s]))
                    page = int(self.pages[s, j // self.page])
                    new = x[self.off[s] + j - past:self.off[s] + hi - past].astype(np.float64)
                    row, old, at = page * self.page + j % self.page, j - lo, (j % self.page) // S
                    j = hi
                    if not 0 <= page < self.n_pages:
                        continue
                    for h in range(self.kv):
                        e = least_exponent(new[:, h])
                        held = int(scale[page, h, at]) - 127
                        if old:
                            e = max(e, held)
                            if e > held:
                                byte[row - old:row, h] = nearest(NUMBERS[byte[row - old:row, h]] * 2.0 ** (held - e))
                        byte[row:row + len(new), h] = nearest(new[:, h] * 2.0**-e)
                        scale[page, h, at] = e + 127
        self.refresh()


def rotate32(x, table, pos, heads, dh, rot, pairs):
    """Rows of x [n, heads*dh] rotated in float32, each product rounded before the sum."""
    y = np.asarray(x, np.float32).reshape(len(pos), heads, dh).copy()
    if rot:
        c, s = (np.ascontiguousarray(table[pos][:, None, :, i]) for i in (0, 1))
        i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
        u, w = y[..., i0].copy(), y[..., i1].copy()
        y[..., i0], y[..., i1] = u * c - w * s, w * c + u * s
    return y


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log of its share, how near the choice came to a border) of one row of logits."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    m = x.max()
    if m == -np.inf:
        return 0, -np.inf, 1.0
    if not temperature > 0 or top_k == 1 or top_p <= 0:
        return int(np.argmax(x)), 0.0, 1.0
    if m == np.inf:
        x, m = np.where(x == np.inf, 0.0, -np.inf), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(np.isneginf(x), 0.0, np.exp((x - m) / float(temperature)))
    w[x == m] = 1.0
    order = np.argsort(-x, kind="stable")
    order = order[:top_k] if 0 < top_k < len(x) else order
    near = 1.0
    if top_p < 1:
        mass = np.cumsum(w[order])
        border = float(top_p) * mass[-1]
        near = float(np.abs(mass / border - 1).min())
        order = order[:1 + int(np.searchsorted(mass, border))]
    if min_p > 0:
        least = min(float(min_p), 1.0)
        near = min(near, float(np.abs(w / least - 1)[w < 1].min(initial=1.0)))
        order = order[(w[order] >= least) | (np.arange(len(order)) == 0)]
    order = np.sort(order)
    mass = np.cumsum(w[order])
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    near = min(near, float(np.abs(mass - u * mass[-1]).min() / mass[-1])) if 0 < u < 1 else near
    live = order[w[order] > 0]
    token = order[min(int(np.searchsorted(mass, u * mass[-1], side="right")), len(order) - 1)]
    token = live[-1] if u >= 1 else token
    return int(token), float(np.log(w[token] / mass[-1])), near


def sample_exact(weights, order, top_k, p, u):
    """The token by whole numbers and fractions: weights of integers, kept ones a prefix of `order`."""
    order = list(order[:top_k] if top_k else order)
    total, run, keep = sum(weights[i] for i in order), 0, []
    for i in order:
        if keep and Fraction(run) >= Fraction(p) * total:
            break
        keep.append(i)
        run += weights[i]
    keep.sort()
    total, run = sum(weights[i] for i in keep), 0
    for i in keep:
        run += weights[i]
        if Fraction(run) > Fraction(u) * total:
            return i
    return keep[-1]
