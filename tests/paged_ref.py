"""The paged K/V cache's operators in float64, from their definitions, with numpy alone.

A `Case` holds what the host knows of a batch and, as plain arrays, the keys and values that its
page tables name: `keys(s)` is the axis that sequence s's tokens look along, prefix first, with a
truth value for every key (false where its page is not there)."""
import numpy as np


def to_bf16_bits(x):
    """Nearest bf16, ties to even, as uint16 (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16_bits(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


class Case:
    """b sequences with n[s] new tokens and length[s] own ones, on a pool whose unused rows hold NaN."""

    def __init__(self, rng, n, length, prefix=0, page=16, kv=2, group=1, dh=32, dtype="f32", max_tok=None,
                 max_own=None, behind=0):
        self.n, self.length, self.prefix = np.asarray(n, int), np.asarray(length, int), prefix
        self.b, self.page, self.kv, self.h, self.dh, self.dtype = len(n), page, kv, kv * group, dh, dtype
        self.off = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.n_tok = int(self.off[-1]) + behind  # rows of the token tensors
        self.max_tok = max_tok or max(1, int(self.n.max(initial=1)))
        self.max_own = int(self.length.max(initial=0)) if max_own is None else max_own
        used, first = -(-self.length // page), -(-prefix // page)
        m = max(1, -(-self.max_own // page))
        self.n_pages = first + int(used.sum()) + 2
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.prefix_pages = order[:first].copy()
        self.pages = np.full((self.b, m), -1, np.int32)
        at = first
        for s in range(self.b):
            self.pages[s, :used[s]] = order[at:at + used[s]]
            at += used[s]
        row = kv * dh
        self.kp = np.full((self.n_pages * page, row), np.nan, np.float32)
        self.vp = np.full((self.n_pages * page, row), np.nan, np.float32)
        for rows in [self.rows(self.prefix_pages, prefix)] + [self.rows(self.pages[s], self.length[s])
                                                              for s in range(self.b)]:
            for pool in (self.kp, self.vp):
                x = rng.standard_normal((len(rows), row)).astype(np.float32)
                pool[rows] = from_bf16_bits(to_bf16_bits(x)) if dtype == "bf16" else x
        self.q = rng.standard_normal((self.n_tok, self.h * dh)).astype(np.float32)

    def rows(self, pages, n):
        j = np.arange(n)
        return pages[j // self.page].astype(np.int64) * self.page + j % self.page

    def keys(self, s):
        """(K [keys, kv, dh], V, there [keys]) along the axis of sequence s."""
        rows = np.concatenate([self.rows(self.prefix_pages, self.prefix), self.rows(self.pages[s], self.length[s])])
        there = (rows >= 0) & (rows < self.n_pages * self.page)
        at = np.where(there, rows, 0)
        return [x[at].astype(np.float64).reshape(-1, self.kv, self.dh) for x in (self.kp, self.vp)] + [there]


def attention(c):
    """(out [n_tok, h*dh], lse [n_tok, h], bound on |out's error|, bound on |lse's|); rows behind the last
    sequence stay NaN.

    The bounds, for 32-bit sums in any order: a score of dh products, q scaled first, is off by at most
    δ = (dh + 4)·2^-24·Σ|q||k|/√dh (dh roundings of products and sums, q's, log2(e)'s and the maximum's
    subtraction on top); the exponential and the final division by 2^-22 together; p by the factor
    1 ± (δ + 2^-22) in numerator and denominator; and the n sums of a row, each a rounding of 2^-24, add
    up as a random walk: 4√n of them, and 8 for joins and rescalings: in all ε = 2δ + (4√n + 24)·2^-24,
    relative to Σ p|v|."""
    d = c.h * c.dh
    out, lse = np.full((c.n_tok, d), np.nan), np.full((c.n_tok, c.h), np.nan)
    tol, tol_lse = np.zeros((c.n_tok, d)), np.zeros((c.n_tok, c.h))
    g = c.h // c.kv
    for s in range(c.b):
        k, v, there = c.keys(s)
        for i in range(c.n[s]):
            t = c.off[s] + i
            sees = there.copy()
            sees[max(c.prefix + c.length[s] - c.n[s] + i + 1, c.prefix):] = False
            for h in range(c.h):
                q = c.q[t, h * c.dh:(h + 1) * c.dh].astype(np.float64)
                kk, vv = k[sees, h // g], v[sees, h // g]
                sl = slice(h * c.dh, (h + 1) * c.dh)
                if len(kk) == 0:
                    out[t, sl], lse[t, h] = 0.0, -np.inf
                    continue
                sc = kk @ q / np.sqrt(c.dh)
                delta = (c.dh + 4) * 2.0**-24 * float((np.abs(kk) @ np.abs(q)).max()) / np.sqrt(c.dh)
                m = sc.max()
                p = np.exp(sc - m)
                l = p.sum()
                with np.errstate(invalid="ignore"):
                    out[t, sl] = (p / l) @ vv
                    eps = 2 * delta + (4 * np.sqrt(len(p)) + 24) * 2.0**-24
                    tol[t, sl] = eps * ((p / l) @ np.abs(vv))
                lse[t, h] = m + np.log(l)
                tol_lse[t, h] = delta + (4 * np.sqrt(len(p)) + 24) * 2.0**-24 + 2.0**-22 * abs(lse[t, h])
    return out, lse, tol, tol_lse


def rotate(x, pos, heads, dh, rot, pairs, theta=10000.0):
    """Rows of x [n, heads*dh] turned by the angles of their positions, in float64."""
    y = np.asarray(x, np.float64).reshape(len(pos), heads, dh).copy()
    half = rot // 2
    if half:
        a = np.asarray(pos, np.float64)[:, None] * theta ** (-2.0 * np.arange(half) / rot)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, half), slice(half, rot))
        u, w = y[..., i0].copy(), y[..., i1].copy()
        y[..., i0], y[..., i1] = u * c - w * s, w * c + u * s
    return y.reshape(len(pos), -1)
