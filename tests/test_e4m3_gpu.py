"""The paged K/V cache in 8 bits on the GPU: appending (elements and scales bit for bit), reading back, and
attention against its definition in float64 on the values that the bytes stand for.  Unused rows hold NaN
and unused scales 255, so that what is read past a sequence's end shows."""
import numpy as np
import pytest

from tests.e4m3_ref import NUMBERS, Case8, nearest, rotate32
from tests.paged_ref import Case, from_bf16_bits, to_bf16_bits
from tests.paged_tiles import ALL, D_HEADS, attention_blocks
from tests.test_paged_gpu import DECODE, POOLED, TAILS, Device, _check, _hip

pytestmark = pytest.mark.gpu


class Device8(Device):
    """A Case8 on the device: the bytes in the pools, and their scales."""

    def __init__(self, ctx, c, **kw):
        from aurora_amd.gpu import GpuBuffer, PagedKvCache

        held, c.dtype = c.dtype, "f32"
        super().__init__(ctx, c, **kw)  # (its pools of floats are replaced)
        c.dtype = held
        self.k.free(), self.v.free()
        self.k, self.v = GpuBuffer.from_slice(ctx, c.kb.ravel()), GpuBuffer.from_slice(ctx, c.vb.ravel())
        self.ks, self.vs = GpuBuffer.from_slice(ctx, c.ks.ravel()), GpuBuffer.from_slice(ctx, c.vs.ravel())
        self.cache = PagedKvCache(self.k, self.v, c.n_pages, c.page, c.kv, c.dh, "e4m3", self.ks, self.vs, c.block)
        from aurora_amd.gpu import PagedMhaKernel
        self.ws.free()
        self.ws_len = PagedMhaKernel.scratch_len(self.cache, self.batch, c.h)
        self.ws = GpuBuffer.from_slice(ctx, np.full(max(1, self.ws_len), np.nan, np.float32))

    def bytes(self):
        c = self.c
        return [b.download().reshape(s.shape) for b, s in ((self.k, c.kb), (self.v, c.vb), (self.ks, c.ks), (self.vs, c.vs))]

    def free(self):
        super().free()
        self.ks.free(), self.vs.free()


def _blocks(page, i):
    """A length of scale blocks for pages of that length, another one for each i."""
    powers = [2**x for x in range(8) if 2**x <= page]
    return powers[i % len(powers)]


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("i,shape", list(enumerate(DECODE + TAILS)))
def test_attention_matches_float64(ctx, i, shape):
    b, n, past, prefix, page, kv, group, dh, _ = shape
    rng = np.random.default_rng(b * 1000 + dh + prefix)
    c = Case8(rng, n, [x + y for x, y in zip(n, past)], prefix, page, kv, group, dh, _blocks(page, i), behind=2)
    dev = Device8(ctx, c, ld_q=c.h * dh + 12, ld_o=c.h * dh + 4)
    dev.attend()
    worst = _check(c, *dev.result())
    print(f"[e4m3] {worst:.3f} of the bound")
    dev.free()


@pytest.mark.parametrize("group", [1, 2, 3])
@pytest.mark.parametrize("dh", [8, 16, 24, 40, 64, 72, 96, 120, 128])
@pytest.mark.parametrize("n,past,prefix", [([1, 0, 1, 1], [0, 9, 62, 500], 0), ([1], [129], 65), ([1, 1, 1], [63, 64, 0], 257),
                                           ([1] * 35, [7 * i % 90 for i in range(35)], 300)])
def test_steps_of_few_rows(ctx, n, past, prefix, dh, group):
    rng = np.random.default_rng(dh + len(n))
    c = Case8(rng, n, [x + y for x, y in zip(n, past)], prefix, 16, 3, group, dh, _blocks(16, dh + group), behind=1)
    dev = Device8(ctx, c, ld_q=c.h * dh + 4)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


@pytest.mark.parametrize("dh", [16, 48, 64, 88, 128])
@pytest.mark.parametrize("b,n,prefix,kv,group", POOLED)
def test_prefix_read_once_for_all(ctx, b, n, prefix, kv, group, dh):
    rng = np.random.default_rng(b + dh)
    toks = [n] * b
    toks[b // 2] = 0
    c = Case8(rng, toks, [x + (5 * i) % 37 for i, x in enumerate(toks)], prefix, 16, kv, group, dh, _blocks(16, b + dh), behind=1)
    dev = Device8(ctx, c, ld_o=c.h * dh + 4)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


@pytest.mark.parametrize("dh", D_HEADS)
@pytest.mark.parametrize("name", ALL)
def test_every_kind_of_item(ctx, name, dh):
    """Batches that reach every kernel, blocks of values up to 2^12 apart."""
    t = ALL[name]
    c = Case8(np.random.default_rng(dh + len(t.n)), t.n, t.length, t.prefix, t.page, t.kv, t.group, dh,
              _blocks(t.page, dh // 8), sizes=(-6, 1))
    dev = Device8(ctx, c)
    dev.attend()
    out, lse = dev.result()
    want, want_lse, tol, tol_lse = attention_blocks(c)
    n = int(c.off[-1])
    assert np.isfinite(out[:n]).all()
    err = np.abs(out[:n] - want[:n]) / np.maximum(tol[:n], 1e-300)
    assert err.max() <= 1.0, f"{err.max()} of the bound"
    e = np.abs(lse[:n] - want_lse[:n]) / tol_lse[:n]
    assert e.max() <= 1.0, f"lse {e.max()} of the bound"
    print(f"[e4m3] {err.max():.3f} of the bound")
    dev.free()


@pytest.mark.parametrize("seed", range(16))
def test_attention_random_batches(ctx, seed):
    rng = np.random.default_rng(100 + seed)
    b, kv, group = int(rng.integers(1, 12)), int(rng.integers(1, 4)), int(rng.choice([1, 1, 2, 3, 5]))
    dh = int(rng.choice([8, 16, 24, 32, 40, 48, 56, 64, 64, 72, 80, 88, 96, 104, 112, 120, 128]))
    n = rng.integers(0, 2 if seed % 2 else int(rng.choice([3, 20, 90])), b)
    n[rng.integers(b)] = max(1, n.max())
    length = n + rng.integers(0, int(rng.choice([2, 40, 400])), b)
    page = int(2 ** rng.integers(0, 8))
    c = Case8(rng, n, length, int(rng.choice([0, 1, 31, 64, 500, 1500])), page, kv, group, dh, _blocks(page, seed),
              max_own=int(length.max()) + int(rng.integers(0, 300)), max_tok=int(n.max()) + int(rng.integers(0, 40)),
              behind=int(rng.integers(0, 3)))
    dev = Device8(ctx, c)
    dev.attend()
    _check(c, *dev.result(), what=f"b={b} n={n} length={length} prefix={c.prefix} page={page} kv={kv} g={group} dh={dh}")
    dev.free()


@pytest.mark.parametrize("n,prefix", [([1, 1, 1], 200), ([40, 70, 1], 90), ([40, 3, 7], 0), ([3, 2, 1], 40)])
def test_pages_that_are_not_there(ctx, n, prefix):
    c = Case8(np.random.default_rng(5), n, [x + 60 for x in n], prefix, 16, 2, 1, 64, 4)
    c.pages[0, 1], c.pages[1, 0], c.pages[2, 2] = -1, c.n_pages, 2**31 - 1
    c.pages[2, :2] = -7
    c.pages[2, 2:] = -1
    if prefix:
        c.prefix_pages[3 % len(c.prefix_pages)], c.prefix_pages[-1] = -2**31, c.n_pages + 5
    dev = Device8(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


def test_rows_without_keys(ctx):
    for prefix in (0, 45):
        c = Case8(np.random.default_rng(2), [6, 1, 1], [2, 0, 9], prefix)
        dev = Device8(ctx, c)
        dev.attend()
        out, lse = dev.result()
        _check(c, out, lse)
        if prefix == 0:
            assert np.all(out[:4] == 0) and np.all(np.isneginf(lse[:4])) and np.all(out[6] == 0)
        dev.free()


@pytest.mark.parametrize("n,prefix,group", [([70, 5], 40, 1), ([9, 33], 0, 3), ([3, 2, 1, 4], 100, 1)])
def test_nan_stays_behind_the_mask(ctx, n, prefix, group):
    """NaN elements, and blocks whose scale is 255, of later tokens reach no earlier one's row."""
    c = Case8(np.random.default_rng(6), n, [x + 4 for x in n], prefix, 8, 2, group, 64, 1)
    own = c.rows(c.pages[0], c.length[0])
    c.vb[own[-2], 3] = 127
    c.kb[own[-1], :64] = 255  # the last token's K of head 0
    page, slot = divmod(int(own[-1]), 8)
    c.vs[page, 1, slot] = 255  # … and its V of head 1, by the scale
    with np.errstate(invalid="ignore"):
        c.refresh()
    c.vp[own[-1], 64:] = np.nan
    dev = Device8(ctx, c)
    dev.attend()
    out, lse = dev.result()
    from tests.paged_ref import attention
    want, want_lse, tol, _ = attention(c)
    rows = [t for t in range(int(c.off[-1])) if t not in (int(c.off[1]) - 1, int(c.off[1]) - 2)]
    assert np.isfinite(want[rows]).all() and np.isfinite(out[rows]).all()
    assert np.all(np.abs(out[rows] - want[rows]) <= tol[rows])
    last = int(c.off[1]) - 1
    assert np.isnan(out[last]).all()
    before = out[last - 1].reshape(c.h, 64)
    assert np.isnan(before[:group, 3]).all() and np.isfinite(np.delete(before, 3, 1)).all()
    dev.free()


@pytest.mark.parametrize("n,prefix", [([1, 1, 1], 400), ([1] * 40, 300), ([90, 70], 60), ([5, 6], 30)])
@pytest.mark.parametrize("k_e,v_e", [(0, -90), (0, 100), (40, 0), (-40, 0)])
def test_scales_of_any_size(ctx, n, prefix, k_e, v_e):
    """Scales far from one: the queries make up for K's."""
    c = Case8(np.random.default_rng(16), n, [x + 20 for x in n], prefix, 16, 1, 1, 64, 8)
    c.ks = np.where(c.ks == 255, 255, c.ks.astype(int) + k_e).astype(np.uint8)
    c.vs = np.where(c.vs == 255, 255, c.vs.astype(int) + v_e).astype(np.uint8)
    with np.errstate(invalid="ignore"):
        c.refresh()
    c.q *= np.float32(2.0**-k_e)
    dev = Device8(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


# ------------------------------------------------------------------ append


# b, new tokens, own tokens before them, prefix, page, block, kv heads, group, d_head, rotated columns, pairs
APPENDS = [
    (1, [1], [0], 0, 16, 16, 1, 1, 8, 8, False),
    (1, [1], [5], 3, 1, 1, 1, 1, 16, 0, False),
    (4, [1] * 4, [0, 1, 15, 16], 32, 16, 16, 4, 1, 32, 32, False),
    (4, [1] * 4, [3, 4, 63, 130], 7, 64, 32, 2, 2, 64, 64, True),
    (3, [40, 0, 17], [0, 9, 30], 0, 16, 4, 3, 1, 48, 16, True),
    (3, [100, 37, 128], [3, 0, 1], 9, 64, 64, 2, 1, 64, 64, False),
    (2, [200, 131], [100, 0], 0, 128, 128, 1, 3, 128, 128, False),  # blocks that four waves share
    (2, [70, 260], [11, 128], 5, 128, 128, 2, 1, 40, 24, False),
    (2, [33, 90], [0, 127], 0, 128, 64, 1, 1, 96, 96, True),
    (5, [2, 3, 1, 7, 5], [6, 5, 7, 0, 9], 0, 8, 8, 5, 1, 24, 8, False),  # blocks that begin with older tokens
    (20, [1] * 20, list(range(20)), 11, 32, 8, 2, 2, 72, 64, False),
    (9, [3] * 9, [5 * i for i in range(9)], 0, 4, 2, 1, 1, 120, 0, False),
]


def _append(ctx, c, dev, q, k, v, table, n_pos, rot, pairs, q_out):
    from aurora_amd.gpu import PagedKvAppendKernel

    d, row = c.h * c.dh, c.kv * c.dh
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, q, d, k, v, row + 4, q_out, d + 4, table, n_pos,
                                            rot, c.h, pairs)


def _table(ctx, n_pos, rot):
    from aurora_amd.gpu import GpuBuffer, RotaryTableKernel

    table = GpuBuffer.zeros(ctx, n_pos * max(rot, 2))
    if rot:
        RotaryTableKernel.new().dispatch_into(ctx, table, n_pos, rot)
    return table, table.download().reshape(n_pos, -1, 2)


def _same_bytes(got, want):
    nan = want & 127 == 127
    assert np.array_equal(got & 127 == 127, nan)
    assert np.array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("b,n,past,prefix,page,block,kv,group,dh,rot,pairs", APPENDS)
@pytest.mark.parametrize("size", [0, 3, -30])
def test_append_gives_the_defined_bytes(ctx, b, n, past, prefix, page, block, kv, group, dh, rot, pairs, size):
    """Elements and scales of an append, for new values about as large as the older ones, larger (blocks that
    hold older tokens take a larger scale) and smaller; all that is not appended to stays as it was."""
    from aurora_amd.gpu import GpuBuffer

    rng = np.random.default_rng(b + dh + page + size + 30)
    c = Case8(rng, n, [x + y for x, y in zip(n, past)], prefix, page, kv, group, dh, block, behind=2)
    dev = Device8(ctx, c)
    n_pos = prefix + int(c.length.max())
    table, t = _table(ctx, n_pos, rot)
    x = [(rng.standard_normal((c.n_tok, w)) * 2.0**s).astype(np.float32) for w, s in ((c.h * dh, 0), (kv * dh, size), (kv * dh, size))]
    pad = [np.pad(a, ((0, 0), (0, w)), constant_values=np.nan) for a, w in zip(x, (0, 4, 4))]
    q, k, v = (GpuBuffer.from_slice(ctx, a.ravel()) for a in pad)
    q_out = GpuBuffer.from_slice(ctx, np.full(c.n_tok * (c.h * dh + 4), 7.5, np.float32))
    _append(ctx, c, dev, q, k, v, table, n_pos, rot, pairs, q_out)
    got = dev.bytes()
    pos = np.zeros(c.n_tok, int)
    for s in range(b):
        pos[c.off[s]:c.off[s + 1]] = prefix + c.length[s] - c.n[s] + np.arange(c.n[s])
    c.append(rotate32(x[1], t, pos, kv, dh, rot, pairs), x[2].reshape(-1, kv, dh))
    for a, w in zip(got, (c.kb, c.vb)):
        _same_bytes(a, w)
    for a, w in zip(got[2:], (c.ks, c.vs)):
        assert np.array_equal(a, w)
    y = q_out.download().reshape(c.n_tok, -1)
    rows = int(c.off[-1])
    assert np.all(y[rows:] == 7.5) and np.all(y[:, c.h * dh:] == 7.5)
    # a rounding of each product and of the sum: three of 2^-24 of a pair's length at most
    want = rotate32(x[0], t, pos, c.h, dh, rot, pairs).reshape(c.n_tok, -1)[:rows]
    assert np.abs(y[:rows, :c.h * dh] - want).max(initial=0) <= 3 * 2.0**-24 * 2 * np.abs(x[0]).max()
    for z in (q, k, v, q_out, table):
        z.free()
    dev.free()


def test_append_token_by_token(ctx):
    """A block filled token by token, each larger than the last, holds what the definition gives in that order,
    and every element is within a step of its scale's e4m3 numbers."""
    from aurora_amd.gpu import GpuBuffer

    rng = np.random.default_rng(3)
    c = Case8(rng, [1, 1], [1, 1], 0, 16, 2, 1, 32, 16, max_own=40)
    c.pages = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    c.n_pages = 6
    c.kb = c.vb = None
    c.kb, c.vb = (np.full((96, 64), 127, np.uint8) for _ in range(2))
    c.ks, c.vs = (np.full((6, 2, 1), 255, np.uint8) for _ in range(2))
    c.kp = c.vp = np.zeros((96, 64), np.float32)
    dev = Device8(ctx, c)
    true = np.zeros((2, 40, 2, 32))
    from aurora_amd.gpu import PagedKvAppendKernel
    for j in range(40):
        x = [(rng.standard_normal((2, 64)) * 1.3**j).astype(np.float32) for _ in range(2)]
        true[:, j] = x[1].reshape(2, 2, 32)
        c.length[:] = j + 1
        dev.len.upload(c.length.astype(np.int32))
        k, v = (GpuBuffer.from_slice(ctx, a.ravel()) for a in x)
        PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, k, v, 64, 0, 0, 0, 0, 0, 0)
        with np.errstate(invalid="ignore"):
            c.append(*(a.reshape(2, 2, 32) for a in x))
        k.free(), v.free()
    got = dev.bytes()
    rows = np.r_[0:40, 48:88]
    for a, w in zip(got, (c.kb, c.vb)):
        _same_bytes(a[rows], w[rows])
    assert np.array_equal(got[2][[0, 1, 2, 3, 4, 5]], c.ks) and np.array_equal(got[3], c.vs)
    for s in range(2):
        for j in range(40):
            row = int(c.pages[s, j // 16]) * 16 + j % 16
            for h in range(2):
                scale = 2.0 ** (int(got[3][row // 16, h, 0]) - 127)
                held = NUMBERS[got[1][row].reshape(2, 32)[h]] * scale
                # half a step of e4m3 once, and below its smallest normal number half a step for each time (at most
                # 16) that the scale grew
                assert np.all(np.abs(held - true[s, j, h]) <= 2.0**-4 * np.abs(true[s, j, h]) * 1.07 + 16 * 2.0**-10 * scale)
    dev.free()


def test_append_of_special_values(ctx):
    """Zeros, subnormals, the largest floats, infinities and NaN."""
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel

    c = Case8(np.random.default_rng(4), [9], [9], 0, 16, 1, 1, 32, 1)
    x = np.ones((9, 32), np.float32)
    x[0] = 0.0
    x[1, :4] = np.inf, -np.inf, np.nan, 3.0
    x[2] = np.nan
    x[3, :3] = 3.4028235e38, -3.4028235e38, 2.9e38
    x[4] = 1e-40
    x[5] = -0.0
    x[6, :3] = 448.0, 464.0, -449.0
    x[7] = 2.0**-117 * 448
    x[8, :5] = 1.75, 1.7500001, 1.8125, 1.9375, -1.0625  # ties, to the even one
    dev = Device8(ctx, c)
    k, v = GpuBuffer.from_slice(ctx, x.ravel()), GpuBuffer.from_slice(ctx, -x.ravel())
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, k, v, 32, 0, 0, 0, 0, 0, 0)
    with np.errstate(invalid="ignore"):
        c.append(x.reshape(9, 1, 32), -x.reshape(9, 1, 32))
    got = dev.bytes()
    for a, w in zip(got, (c.kb, c.vb)):
        _same_bytes(a, w)
    assert np.array_equal(got[2], c.ks) and np.array_equal(got[3], c.vs)
    row = int(c.rows(c.pages[0], 9)[3])
    assert NUMBERS[got[0][row, 0]] == 448 and got[2].reshape(-1)[row] == 127 + 119
    dev.free(), k.free(), v.free()


def test_append_drops_what_has_no_place(ctx):
    """Tokens in front of the sequence's first, rows of pages that are not there: nothing of them is written."""
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel

    rng = np.random.default_rng(7)
    c = Case8(rng, [30, 5, 20], [20, 5, 50], 0, 8, 2, 1, 32, 4)
    c.pages[2, 5], c.pages[1, 0], c.pages[0, 1] = -3, c.n_pages, 2**31 - 1
    dev = Device8(ctx, c)
    x = [rng.standard_normal((c.n_tok, 64)).astype(np.float32) * 4 for _ in range(2)]
    k, v = (GpuBuffer.from_slice(ctx, a.ravel()) for a in x)
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, k, v, 64, 0, 0, 0, 0, 0, 0)
    with np.errstate(invalid="ignore"):
        c.append(*(a.reshape(-1, 2, 32) for a in x))
    got = dev.bytes()
    for a, w in zip(got, (c.kb, c.vb)):
        _same_bytes(a, w)
    assert np.array_equal(got[2], c.ks) and np.array_equal(got[3], c.vs)
    dev.free(), k.free(), v.free()


# ------------------------------------------------------------------ read back


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("b,length,prefix,page,kv,dh,first,count", [
    (1, [1], 0, 1, 1, 8, 0, 1),
    (3, [0, 17, 64], 33, 16, 3, 24, 0, 97),
    (3, [0, 17, 64], 33, 16, 3, 24, 30, 40),     # across the prefix's end
    (2, [100, 31], 0, 64, 2, 128, 7, 90),
    (5, [3, 300, 1, 77, 299], 77, 8, 16, 64, 0, 377),
    (2, [5, 9], 200, 32, 5, 120, 100, 50),       # of the prefix alone
])
def test_read_back(ctx, dtype, b, length, prefix, page, kv, dh, first, count):
    from aurora_amd.gpu import GpuBuffer, PagedKvReadKernel

    rng = np.random.default_rng(b + dh)
    n = [min(1, x) for x in length]
    c = (Case8(rng, n, length, prefix, page, kv, 1, dh, _blocks(page, dh // 8)) if dtype == "e4m3"
         else Case(rng, n, length, prefix, page, kv, 1, dh, dtype))
    if b > 2:
        c.pages[1, 1] = -1  # a page that is not there
    dev = (Device8 if dtype == "e4m3" else Device)(ctx, c)
    row = kv * dh
    ld = row + 4
    outs = [GpuBuffer.from_slice(ctx, np.full(b * count * ld, 7.5, np.float32)) for _ in range(2)]
    PagedKvReadKernel.new().dispatch_into(ctx, dev.cache, dev.batch, outs[0], outs[1], ld, first, count)
    for out, pool in zip(outs, (0, 1)):
        got = out.download().reshape(b, count, ld)
        assert np.all(got[..., row:] == 7.5)
        want = np.zeros((b, count, row))
        for s in range(b):
            x, there = c.keys(s)[pool], c.keys(s)[2]
            x = np.where(there[:, None, None], x, 0.0).reshape(len(x), row)[first:first + count]
            want[s, :len(x)] = x
        assert np.array_equal(got[..., :row], want)
    # one of the two alone
    outs[0].zero()
    PagedKvReadKernel.new().dispatch_into(ctx, dev.cache, dev.batch, outs[0], 0, ld, first, count)
    got = outs[0].download().reshape(b, count, ld)
    assert np.all(got[..., row:] == 0)
    for out in outs:
        out.free()
    dev.free()


# ------------------------------------------------------------------ a run of them


@pytest.mark.parametrize("dh,kv,group,block", [(64, 2, 2, 16), (32, 3, 1, 4)])
def test_prompt_and_steps(ctx, dh, kv, group, block):
    """A shared prefix and prompts are appended and attended to, then steps of one token; each attention is what
    float64 makes of the rows that reading back gives, and these are near the values appended."""
    from aurora_amd.gpu import (GpuBuffer, PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedKvReadKernel, PagedMhaKernel,
                                RotaryTableKernel)

    rng = np.random.default_rng(11)
    h, page, P, prompts, steps = kv * group, 16, 37, [20, 9, 33], 5
    d, row, b = h * dh, kv * dh, len(prompts)
    cache = PagedKvCache.zeros(ctx, 24, page, kv, dh, "e4m3", scale_len=block)
    most = max(prompts) + steps
    n_pos = P + most
    table = GpuBuffer.zeros(ctx, n_pos * dh)
    RotaryTableKernel.new().dispatch_into(ctx, table, n_pos, dh)
    pages = rng.permutation(24).astype(np.int32)
    prefix = GpuBuffer.from_slice(ctx, pages[:3])
    m = -(-most // page)
    own = GpuBuffer.from_slice(ctx, pages[3:3 + b * m])
    i32 = lambda x: GpuBuffer.from_slice(ctx, np.asarray(x, np.int32))  # noqa: E731
    append, attend, read = PagedKvAppendKernel.new(), PagedMhaKernel.new(), PagedKvReadKernel.new()
    f = lambda n, w: rng.standard_normal((n, w)).astype(np.float32)  # noqa: E731
    up = lambda x: GpuBuffer.from_slice(ctx, x.ravel())  # noqa: E731

    k0, v0 = f(P, row), f(P, row)
    first = PagedBatch(i32([0, P]), i32([P]), prefix, 1, 3, P, P, P)
    append.dispatch_into(ctx, cache, first, 0, 0, up(k0), up(v0), row, 0, 0, table, n_pos, dh, 0)
    held_v = [[v0] for _ in range(b)]
    length = np.zeros(b, int)
    for step in range(1 + steps):
        n = np.array(prompts) if step == 0 else np.ones(b, int)
        length += n
        off = np.concatenate([[0], np.cumsum(n)])
        t = int(off[-1])
        q, k, v = f(t, d), f(t, row), f(t, row)
        for s in range(b):
            held_v[s].append(v[off[s]:off[s + 1]])
        batch = PagedBatch(i32(off), i32(length), own, b, m, t, int(n.max()), most, prefix, 3, P)
        bq, out = up(q), GpuBuffer.zeros(ctx, t * d)
        append.dispatch_into(ctx, cache, batch, bq, d, up(k), up(v), row, bq, d, table, n_pos, dh, h)
        ws_len = PagedMhaKernel.scratch_len(cache, batch, h)
        attend.dispatch_into(ctx, cache, batch, bq, d, out, d, 0, GpuBuffer.empty(ctx, max(1, ws_len)), ws_len, h)
        ko, vo = (GpuBuffer.empty(ctx, b * (P + most) * row) for _ in range(2))
        read.dispatch_into(ctx, cache, batch, ko, vo, row, 0, P + most)
        ko, vo = (x.download().reshape(b, P + most, kv, dh).astype(np.float64) for x in (ko, vo))
        qr, got = bq.download().reshape(t, h, dh).astype(np.float64), out.download().reshape(t, h, dh)
        for s in range(b):
            true = np.concatenate(held_v[s]).reshape(-1, kv, dh)
            keys = P + length[s]
            assert np.all(vo[s, keys:] == 0) and np.all(ko[s, keys:] == 0)
            # half a step of e4m3, or of the smallest numbers of a scale that a value below 8 gives (2^-5·2^-10)
            assert np.all(np.abs(vo[s, :keys] - true) <= 2.0**-4 * 1.07 * np.abs(true) + 2.0**-10)
            for i in range(int(n[s])):
                sees = keys - int(n[s]) + i + 1
                for head in range(h):
                    sc = ko[s, :sees, head // group] @ qr[off[s] + i, head] / np.sqrt(dh)
                    p = np.exp(sc - sc.max())
                    want = p @ vo[s, :sees, head // group] / p.sum()
                    np.testing.assert_allclose(got[off[s] + i, head], want, rtol=0, atol=2e-5)
    cache.free()


def test_step_captured_into_a_graph(ctx):
    """Append and attention of a decode step captured once, replayed as lengths grow: as the eager step, bit for bit."""
    from aurora_amd._lib import load
    from aurora_amd.gpu import GpuBuffer

    import ctypes

    hip, stream = _hip(), load().aur_stream(ctx.ptr)
    rng = np.random.default_rng(9)
    c = Case8(rng, [1] * 6, [20, 1, 33, 7, 64, 5], 300, 16, 2, 2, 64, 8, max_own=80)
    c.pages[:] = rng.permutation(6 * 5).reshape(6, 5)
    c.n_pages = max(c.n_pages, 30 + len(c.prefix_pages))
    c.prefix_pages = np.arange(30, 30 + len(c.prefix_pages)).astype(np.int32)
    rows = c.n_pages * 16
    c.kb, c.vb = (nearest(rng.standard_normal((rows, 128)) * 64) for _ in range(2))
    c.ks, c.vs = (np.full((c.n_pages, 2, 2), 121, np.uint8) for _ in range(2))
    c.refresh()
    dev, other = Device8(ctx, c), Device8(ctx, c)
    table, _ = _table(ctx, 400, 64)
    bufs = {}
    for name, w in (("q", 256), ("k", 128 + 4), ("v", 128 + 4)):
        bufs[name] = GpuBuffer.zeros(ctx, 6 * w)
    q_out = GpuBuffer.zeros(ctx, 6 * 260)

    def step(on):
        _append(ctx, c, on, bufs["q"], bufs["k"], bufs["v"], table, 400, 64, False, q_out)
        on.attend()

    for i in range(3):
        for name, b in bufs.items():
            b.upload(rng.standard_normal(b.len).astype(np.float32) * (1 + 3 * i))
        length = np.array([20, 1, 33, 7, 64, 5], np.int32) + i
        dev.len.upload(length), other.len.upload(length)
        if i == 0:
            graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
            ctx.sync()
            assert hip.hipStreamBeginCapture(stream, 1) == 0  # hipStreamCaptureModeThreadLocal
            try:
                step(dev)
            finally:
                assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
        assert hip.hipGraphLaunch(ex, stream) == 0
        ctx.sync()
        step(other)
        for a, w in zip(dev.bytes(), other.bytes()):
            assert np.array_equal(a, w)
        for a, w in zip(dev.result(), other.result()):
            assert np.array_equal(a, w) and np.isfinite(a).all()
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    dev.free(), other.free()
