"""The paged K/V cache on the GPU: appending with the position rotation, and the attention of
sequences that share a prefix, against their definitions in float64 (tests/paged_ref.py, which also
derives the attention's error bounds).  Unused rows of every pool hold NaN, so that a key read past a
sequence's end shows."""
import ctypes

import numpy as np
import pytest

from tests.attn_ref import causal_attention_f64
from tests.paged_ref import Case, attention, from_bf16_bits, rotate, to_bf16_bits

pytestmark = pytest.mark.gpu

U32 = 2.0**-24  # a rounding to 32 bits, relative


class Device:
    """A case's tensors on the device, and the calls."""

    def __init__(self, ctx, c, lse=True, ld_q=None, ld_o=None):
        from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvCache, PagedMhaKernel

        self.ctx, self.c = ctx, c
        d = c.h * c.dh
        self.ld_q, self.ld_o = ld_q or d, ld_o or d
        up = lambda x: GpuBuffer.from_slice(ctx, x)  # noqa: E731
        pool = (lambda x: up(to_bf16_bits(x).ravel())) if c.dtype == "bf16" else (lambda x: up(x.ravel()))
        self.k, self.v = pool(c.kp), pool(c.vp)
        self.off, self.len = up(c.off), up(c.length.astype(np.int32))
        self.pages, self.prefix = up(c.pages.ravel()), up(c.prefix_pages if c.prefix else np.zeros(1, np.int32))
        qs = np.full((c.n_tok, self.ld_q), np.nan, np.float32)
        qs[:c.off[-1], :d] = c.q[:c.off[-1]]  # rows behind the last sequence hold NaN, like the padding of the others
        self.q = up(qs.ravel())
        self.out = GpuBuffer.from_slice(ctx, np.full(c.n_tok * self.ld_o, 7.5, np.float32))
        self.lse = GpuBuffer.from_slice(ctx, np.full(c.n_tok * c.h, 7.5, np.float32)) if lse else 0
        self.cache = PagedKvCache(self.k, self.v, c.n_pages, c.page, c.kv, c.dh, c.dtype)
        self.batch = PagedBatch(self.off, self.len, self.pages, c.b, c.pages.shape[1], c.n_tok, c.max_tok, c.max_own,
                                self.prefix, len(c.prefix_pages), c.prefix)
        self.ws_len = PagedMhaKernel.scratch_len(self.cache, self.batch, c.h)
        # the scratch is exactly as long as asked for, and not clean
        self.ws = GpuBuffer.from_slice(ctx, np.full(max(1, self.ws_len), np.nan, np.float32))

    def attend(self, ctx=None, ws=None):
        from aurora_amd.gpu import PagedMhaKernel

        PagedMhaKernel.new().dispatch_into(ctx or self.ctx, self.cache, self.batch, self.q, self.ld_q, self.out,
                                           self.ld_o, self.lse, ws or self.ws, self.ws_len, self.c.h)

    def result(self):
        out = self.out.download().reshape(self.c.n_tok, self.ld_o)
        return out, self.lse.download().reshape(self.c.n_tok, self.c.h) if self.lse else None

    def free(self):
        for x in (self.k, self.v, self.off, self.len, self.pages, self.prefix, self.q, self.out, self.lse, self.ws):
            if x:
                x.free()


def _check(c, out, lse, what=""):
    want, want_lse, tol, tol_lse = attention(c)
    d, n = c.h * c.dh, int(c.off[-1])
    assert np.all(out[n:] == 7.5) and np.all(out[:, d:] == 7.5), f"{what}: rows or columns that are none were written"
    got, want, tol = out[:n, :d], want[:n], tol[:n]
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)), what
    assert np.array_equal(np.isnan(want), np.isnan(got)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    err = np.abs(got[fine] - want[fine]) / np.maximum(tol[fine], 1e-300)
    worst = float(err.max(initial=0))
    assert worst <= 1.0, f"{what}: {worst} of the bound"
    if lse is not None:
        assert np.all(lse[n:] == 7.5)
        none = np.isneginf(want_lse[:n])
        assert np.array_equal(none, np.isneginf(lse[:n])), what
        e = np.abs(lse[:n][~none] - want_lse[:n][~none]) / tol_lse[:n][~none]
        assert e.max(initial=0) <= 1.0, f"{what}: lse {e.max()} of the bound"
    return worst


# b, new tokens, own tokens before them, prefix, page_len, kv heads, group, d_head, type
DECODE = [
    (1, [1], [0], 0, 16, 1, 1, 8, "f32"),          # one key in all
    (1, [1], [0], 1, 1, 1, 1, 16, "f32"),          # pages of one row
    (1, [1], [4000], 0, 64, 2, 1, 64, "f32"),      # one long axis
    (4, [1] * 4, [0, 1, 31, 30], 32, 16, 4, 1, 32, "f32"),
    (4, [1] * 4, [5, 0, 130, 64], 33, 8, 3, 2, 48, "bf16"),
    (3, [1, 0, 1], [127, 60, 128], 127, 16, 2, 6, 40, "f32"),  # a sequence without new tokens
    (5, [1] * 5, [7, 100, 3, 1, 299], 777, 32, 2, 4, 128, "f32"),
    (5, [1] * 5, [7, 100, 3, 1, 299], 777, 32, 2, 1, 96, "bf16"),
    (33, [1] * 33, list(range(33)), 515, 4, 1, 1, 64, "f32"),
    (70, [1] * 70, [3 * i % 50 for i in range(70)], 200, 64, 2, 1, 64, "bf16"),
    (9, [1] * 9, [1000] * 9, 0, 1024, 1, 1, 72, "f32"),  # no prefix: only own keys, pages longer than they
    (2, [1, 1], [40, 2], 3000, 16, 1, 12, 24, "bf16"),
    (17, [1] * 17, [9] * 17, 65, 2, 5, 1, 56, "f32"),
]
TAILS = [
    (1, [40], [0], 0, 16, 2, 1, 64, "f32"),        # a prompt: plain causal attention
    (1, [200], [0], 0, 64, 1, 1, 32, "bf16"),
    (3, [5, 1, 17], [0, 30, 2], 50, 16, 2, 1, 64, "f32"),
    (3, [64, 65, 63], [0, 1, 100], 130, 32, 1, 1, 64, "f32"),
    (2, [33, 40], [10, 0], 100, 8, 2, 3, 48, "bf16"),
    (4, [12, 0, 3, 20], [0, 5, 1, 0], 0, 4, 1, 2, 80, "f32"),
    (2, [70, 9], [300, 0], 257, 128, 2, 2, 128, "f32"),
    (2, [70, 9], [300, 0], 257, 128, 2, 2, 104, "bf16"),
    (3, [100, 37, 128], [3, 0, 1], 333, 16, 1, 1, 16, "f32"),
    (6, [2, 2, 3, 2, 1, 2], [9, 0, 77, 5, 6, 40], 600, 16, 2, 1, 64, "bf16"),
    (1, [129], [70], 65, 16, 1, 4, 64, "bf16"),
    (16, [4] * 16, [3] * 16, 300, 16, 1, 1, 8, "f32"),
]


@pytest.mark.parametrize("b,n,past,prefix,page,kv,group,dh,dtype", DECODE + TAILS)
def test_attention_matches_float64(ctx, b, n, past, prefix, page, kv, group, dh, dtype):
    rng = np.random.default_rng(b * 1000 + dh + prefix)
    c = Case(rng, n, [x + y for x, y in zip(n, past)], prefix, page, kv, group, dh, dtype, behind=2)
    dev = Device(ctx, c, ld_q=c.h * dh + 12, ld_o=c.h * dh + 4)
    dev.attend()
    worst = _check(c, *dev.result())
    print(f"[paged] {worst:.3f} of the bound")
    dev.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 3])
@pytest.mark.parametrize("dh", [8, 16, 24, 40, 64, 72, 96, 120, 128])
@pytest.mark.parametrize("n,past,prefix", [([1, 0, 1, 1], [0, 9, 62, 500], 0), ([1], [129], 65), ([1, 1, 1], [63, 64, 0], 257),
                                           ([1] * 35, [7 * i % 90 for i in range(35)], 300)])
def test_steps_of_few_rows(ctx, n, past, prefix, dh, group, dtype):
    """One new token a sequence, few heads on the same keys: the lengths around a wave's step."""
    rng = np.random.default_rng(dh + len(n))
    c = Case(rng, n, [x + y for x, y in zip(n, past)], prefix, 16, 3, group, dh, dtype, behind=1)
    dev = Device(ctx, c, ld_q=c.h * dh + 4)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


POOLED = [  # sequences, tokens of each, prefix, kv heads, group: enough of them that the prefix is read once for all
    (20, 1, 1300, 3, 1),   # 20 rows on the prefix
    (9, 1, 2500, 4, 3),
    (40, 1, 900, 2, 1),    # 40
    (40, 1, 900, 2, 2),
    (23, 1, 1601, 2, 4),
    (30, 1, 1201, 2, 5),   # 150
    (90, 1, 401, 2, 3),    # 270: prefix items of their own launch
    (21, 3, 1177, 3, 2),   # several tokens
    (12, 9, 2001, 3, 3),   # 27 own rows
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dh", [16, 48, 64, 88, 128])
@pytest.mark.parametrize("b,n,prefix,kv,group", POOLED)
def test_prefix_read_once_for_all(ctx, b, n, prefix, kv, group, dh, dtype):
    rng = np.random.default_rng(b + dh)
    toks = [n] * b
    toks[b // 2] = 0  # a sequence that waits
    c = Case(rng, toks, [x + (5 * i) % 37 for i, x in enumerate(toks)], prefix, 16, kv, group, dh, dtype, behind=1)
    dev = Device(ctx, c, ld_o=c.h * dh + 4)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


@pytest.mark.parametrize("seed", range(12))
def test_attention_random_batches(ctx, seed):
    rng = np.random.default_rng(seed)
    b, kv, group = int(rng.integers(1, 12)), int(rng.integers(1, 4)), int(rng.choice([1, 1, 2, 3, 5]))
    dh = int(rng.choice([8, 16, 24, 32, 40, 48, 56, 64, 64, 72, 80, 88, 96, 104, 112, 120, 128]))
    n = rng.integers(0, 2 if seed % 2 else int(rng.choice([3, 20, 90])), b)
    n[rng.integers(b)] = max(1, n.max())
    length = n + rng.integers(0, int(rng.choice([2, 40, 400])), b)
    c = Case(rng, n, length, int(rng.choice([0, 1, 31, 64, 500, 1500])), int(2 ** rng.integers(0, 8)), kv, group, dh,
             ["f32", "bf16"][seed % 3 == 0], max_own=int(length.max()) + int(rng.integers(0, 300)),
             max_tok=int(n.max()) + int(rng.integers(0, 40)), behind=int(rng.integers(0, 3)))
    dev = Device(ctx, c)
    dev.attend()
    _check(c, *dev.result(), what=f"b={b} n={n} length={length} prefix={c.prefix} page={c.page} kv={kv} g={group} dh={dh}")
    dev.free()


def test_attention_without_lse(ctx):
    c = Case(np.random.default_rng(1), [1, 1, 1], [50, 60, 70], 300)
    dev = Device(ctx, c, lse=False)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


def test_rows_without_keys(ctx):
    """Fewer own tokens than new ones: the first rows see the prefix alone, or nothing."""
    for prefix in (0, 45):
        c = Case(np.random.default_rng(2), [6, 1, 1], [2, 0, 9], prefix)
        dev = Device(ctx, c)
        dev.attend()
        out, lse = dev.result()
        _check(c, out, lse)
        if prefix == 0:
            assert np.all(out[:4] == 0) and np.all(np.isneginf(lse[:4])) and np.all(out[6] == 0)
        dev.free()


@pytest.mark.parametrize("dtype,n,prefix", [("f32", [1, 1, 1], 200), ("bf16", [1, 1, 1], 200), ("f32", [40, 70, 1], 90),
                                            ("bf16", [40, 3, 7], 0)])
def test_pages_that_are_not_there(ctx, dtype, n, prefix):
    """Page numbers outside the pool take their keys out, of prefix and own ones."""
    rng = np.random.default_rng(5)
    c = Case(rng, n, [x + 60 for x in n], prefix, 16, 2, 1, 64, dtype)
    c.pages[0, 1], c.pages[1, 0], c.pages[2, 2] = -1, c.n_pages, 2**31 - 1
    c.pages[2, :2] = -7  # this sequence keeps its third page and its last rows only …
    c.pages[2, 2:] = -1  # … or nothing of its own at all
    if prefix:
        c.prefix_pages[3], c.prefix_pages[-1] = -2**31, c.n_pages + 5
    dev = Device(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,prefix,group", [([70, 5], 40, 1), ([9, 33], 0, 3), ([3, 2, 1, 4], 100, 1)])
def test_infinities_stay_behind_the_mask(ctx, dtype, n, prefix, group):
    """An infinity or NaN in K or V of a later token reaches no earlier one's row."""
    rng = np.random.default_rng(6)
    c = Case(rng, n, [x + 4 for x in n], prefix, 8, 2, group, 64, dtype)
    s, own = 0, c.rows(c.pages[0], c.length[0])
    at = own[c.length[s] - c.n[s] + c.n[s] // 2]
    c.vp[at, 3], c.vp[at, 70] = np.inf, np.nan
    c.vp[own[-1], 5] = -np.inf
    c.kp[own[-1], :64] = np.nan  # the last token's K of head 0
    c.kp[own[-1], 64:] = 3e38
    dev = Device(ctx, c)
    dev.attend()
    out, lse = dev.result()
    last = int(c.off[1]) - 1  # this row sees them all; what it gets is not a number, or not finite
    want, want_lse, tol, _ = attention(c)
    rows = [t for t in range(int(c.off[-1])) if t != last]
    got, want, tol = out[rows], want[rows], tol[rows]
    fine = np.isfinite(want)
    assert fine.sum() > 0 and np.array_equal(fine, np.isfinite(got))
    assert np.all(np.abs(got[fine] - want[fine]) <= tol[fine])
    assert np.all(np.abs(lse[rows] - want_lse[rows]) < 1e-4)
    g = c.h // c.kv
    assert np.all(np.isnan(out[last, :g * 64]))  # head 0's K is NaN
    dev.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_infinities_that_single_tokens_see(ctx, dtype, group):
    """Infinities and NaN among the keys of a step give what the formula gives, and only where they are seen."""
    c = Case(np.random.default_rng(15), [1] * 5, [90, 40, 130, 70, 20], 40, 8, 2, group, 64, dtype)
    own = [c.rows(c.pages[s], c.length[s]) for s in range(5)]
    c.vp[own[0][5], 3], c.vp[own[0][80], 70] = np.inf, -np.inf
    c.vp[own[1][39], 9] = np.nan
    c.kp[own[2][100], 2] = np.inf  # the query's sign decides: NaN, or a key without weight
    c.kp[own[3][0], 64:] = np.nan
    dev = Device(ctx, c)
    dev.attend()
    out, lse = dev.result()
    with np.errstate(all="ignore"):
        want, _, tol, _ = attention(c)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(out)) and np.array_equal(np.isnan(want), np.isnan(out))
    assert np.array_equal(out[np.isinf(want)], want[np.isinf(want)])
    bounded = fine & np.isfinite(tol)  # (an infinite key without weight leaves its row no bound)
    assert bounded[4].all() and bounded[0].sum() == c.h * 64 - 2 * group
    assert np.all(np.abs(out[bounded] - want[bounded]) <= tol[bounded])
    dev.free()


def test_large_scores_and_small_ones(ctx):
    """Scores far apart (±10^3, where the softmax is a single key) and all −∞."""
    rng = np.random.default_rng(8)
    c = Case(rng, [1, 2], [30, 40], 100, 16, 1, 1, 64)
    c.kp *= 300
    dev = Device(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()
    c.q[:] = np.abs(c.q)
    c.kp[:] = -np.inf
    dev = Device(ctx, c)
    dev.attend()
    out, lse = dev.result()
    assert np.all(out == 0) and np.all(np.isneginf(lse))
    dev.free()


@pytest.mark.parametrize("n,prefix,dtype", [([1, 1, 1], 400, "f32"), ([1] * 40, 300, "f32"), ([1] * 40, 300, "bf16"),
                                            ([90, 70], 60, "f32"), ([90, 70], 60, "bf16"), ([300], 0, "f32")])
@pytest.mark.parametrize("vs,ks", [(2.0**-100, 1.0), (2.0**100, 1.0), (1.0, 2.0**40), (1.0, 2.0**-40)])
def test_values_of_any_size(ctx, n, prefix, dtype, vs, ks):
    """V of any size, and columns of K far larger or smaller than the others whose queries make up for
    it: nothing is lost beside a larger neighbour."""
    rng = np.random.default_rng(16)
    c = Case(rng, n, [x + 20 for x in n], prefix, 16, 1, 1, 64, dtype)
    c.vp[:, ::2] *= np.float32(vs)
    c.kp[:, 1::3] *= np.float32(ks)
    c.q[:, 1::3] /= np.float32(ks)
    dev = Device(ctx, c)
    dev.attend()
    _check(c, *dev.result())
    dev.free()


def _hip():
    hip = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    hip.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    hip.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
    for f in (hip.hipGraphExecDestroy, hip.hipGraphDestroy):
        f.argtypes = [vp]
    hip.hipGraphLaunch.argtypes = [vp, vp]
    return hip


def test_step_captured_into_a_graph(ctx):
    """One decode step (append and attention) captured once and replayed as lengths and pages grow on
    the device, with eager calls in between: every replay equals the eager step bit for bit."""
    from aurora_amd._lib import load
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel, RotaryTableKernel

    hip, stream = _hip(), load().aur_stream(ctx.ptr)
    rng = np.random.default_rng(9)
    steps = 4
    c = Case(rng, [1] * 6, [20, 1, 33, 7, 64, 5], 300, 16, 2, 2, 64, "bf16", max_own=80)
    c.pages[:] = rng.permutation(6 * 5).reshape(6, 5)  # every sequence has its pages for all steps
    c.n_pages = max(c.n_pages, 30 + len(c.prefix_pages))
    c.prefix_pages[:] = 30 + np.arange(len(c.prefix_pages))
    c.kp, c.vp = (rng.standard_normal((c.n_pages * 16, 128)).astype(np.float32) for _ in range(2))
    new = [rng.standard_normal((3, 6, 256)).astype(np.float32) for _ in range(steps)]

    def build():
        dev = Device(ctx, c)
        dev.kn, dev.vn = GpuBuffer.zeros(ctx, 6 * 128), GpuBuffer.zeros(ctx, 6 * 128)
        dev.table = GpuBuffer.empty(ctx, 380 * 64)
        RotaryTableKernel.new().dispatch_into(ctx, dev.table, 380, 64)
        return dev

    def feed(dev, s):
        dev.q.upload(new[s][0].ravel())
        dev.kn.upload(new[s][1, :, :128].ravel())
        dev.vn.upload(new[s][2, :, :128].ravel())
        dev.len.upload(c.length + s)

    def step(dev):
        PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, dev.q, 256, dev.kn, dev.vn, 128, dev.q, 256,
                                                dev.table, 380, 64, 4)
        dev.attend()

    eager, replayed = build(), build()
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(stream, 1) == 0  # hipStreamCaptureModeThreadLocal
    try:
        step(replayed)
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    try:
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for s in range(steps):
            feed(eager, s)
            feed(replayed, s)
            step(eager)
            ctx.sync()
            assert hip.hipGraphLaunch(exe, stream) == 0
            ctx.sync()
            for x, y in zip(eager.result(), replayed.result()):
                assert np.array_equal(x, y), s
            assert np.array_equal(eager.k.download(), replayed.k.download()), s
    finally:
        if exe.value:
            hip.hipGraphExecDestroy(exe)
        if graph.value:
            hip.hipGraphDestroy(graph)
        for dev in (eager, replayed):
            for x in (dev.kn, dev.vn, dev.table):
                x.free()
            dev.free()


def test_two_contexts_at_once_and_the_same_bits(ctx):
    """Calls on two streams with a scratch each, and a call again, give the same bits."""
    from aurora_amd.gpu import GpuBuffer, GpuContext

    c = Case(np.random.default_rng(10), [1] * 20, list(range(1, 201, 10)), 2000, 64, 4, 1, 64)
    dev = Device(ctx, c)
    dev.attend()
    first = dev.result()
    with GpuContext.new(0) as other:
        dev2 = Device(other, c)
        other.sync()
        for _ in range(5):
            dev.attend()
            dev2.attend()
        for got in (dev.result(), dev2.result()):
            for x, y in zip(first, got):
                assert np.array_equal(x, y)
        dev2.free()
    dev.free()


def test_pool_beyond_32_bit_offsets(ctx):
    """Pages whose elements start beyond 2^32 bytes and 2^31 elements."""
    from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedMhaKernel

    kv, dh, page = 16, 128, 256
    row = kv * dh
    n_pages = (2**31 + 2**28) // (page * row)  # bf16: 4.8 GB a pool
    rng = np.random.default_rng(11)
    c = Case(rng, [300], [300], 0, page, kv, 1, dh, "bf16")
    pages = np.array([[n_pages - 1, n_pages - 3]], np.int32)
    cache = PagedKvCache(GpuBuffer.empty(ctx, n_pages * page * row, np.uint16),
                         GpuBuffer.empty(ctx, n_pages * page * row, np.uint16), n_pages, page, kv, dh, "bf16")
    up = lambda x: GpuBuffer.from_slice(ctx, x)  # noqa: E731
    k, v = rng.standard_normal((2, 300, row)).astype(np.float32)
    bufs = [up(np.array([0, 300], np.int32)), up(np.array([300], np.int32)), up(pages.ravel()), up(k.ravel()), up(v.ravel()),
            up(c.q.ravel()), GpuBuffer.empty(ctx, 300 * row)]
    off, length, pg, bk, bv, bq, out = bufs
    batch = PagedBatch(off, length, pg, 1, 2, 300, 300, 300)
    PagedKvAppendKernel.new().dispatch_into(ctx, cache, batch, 0, 0, bk, bv, row, 0, 0, 0, 0, 0, kv)
    n = PagedMhaKernel.scratch_len(cache, batch, kv)
    ws = GpuBuffer.empty(ctx, max(1, n))
    PagedMhaKernel.new().dispatch_into(ctx, cache, batch, bq, row, out, row, 0, ws, n, kv)
    got = out.download().reshape(300, row)
    c.kp, c.vp = (from_bf16_bits(to_bf16_bits(x)) for x in (k, v))
    c.pages, c.n_pages = np.array([[0, 1]], np.int32), 2
    want, _, tol, _ = attention(c)
    assert np.all(np.abs(got - want) <= tol)
    for x in bufs + [ws]:
        x.free()
    cache.free()


@pytest.mark.parametrize("n,group", [(1, 1), (1, 2), (1, 16), (3, 4)])
def test_step_beyond_32_bit_offsets(ctx, n, group):
    """The same for items of few rows."""
    from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedMhaKernel

    kv, dh, page, own = 16, 128, 256, 300
    row, d = kv * dh, kv * dh * group
    n_pages = (2**31 + 2**28) // (page * row)
    rng = np.random.default_rng(16)
    c = Case(rng, [n], [own], 0, page, kv, group, dh, "bf16")
    cache = PagedKvCache(GpuBuffer.empty(ctx, n_pages * page * row, np.uint16),
                         GpuBuffer.empty(ctx, n_pages * page * row, np.uint16), n_pages, page, kv, dh, "bf16")
    up = lambda x: GpuBuffer.from_slice(ctx, x)  # noqa: E731
    k, v = rng.standard_normal((2, own, row)).astype(np.float32)
    bufs = [up(np.array([0, own, 0, n], np.int32)), up(np.array([own], np.int32)),
            up(np.array([n_pages - 1, n_pages - 3], np.int32)), up(k.ravel()), up(v.ravel()), up(c.q.ravel()),
            GpuBuffer.empty(ctx, n * d)]
    off, length, pg, bk, bv, bq, out = bufs
    PagedKvAppendKernel.new().dispatch_into(ctx, cache, PagedBatch(off, length, pg, 1, 2, own, own, own), 0, 0, bk, bv,
                                            row, 0, 0, 0, 0, 0, kv)
    batch = PagedBatch(off.ptr + 8, length, pg, 1, 2, n, n, own)
    ws_len = PagedMhaKernel.scratch_len(cache, batch, c.h)
    ws = GpuBuffer.empty(ctx, max(1, ws_len))
    PagedMhaKernel.new().dispatch_into(ctx, cache, batch, bq, d, out, d, 0, ws, ws_len, c.h)
    c.kp, c.vp = (from_bf16_bits(to_bf16_bits(x)) for x in (k, v))
    c.pages, c.n_pages = np.array([[0, 1]], np.int32), 2
    want, _, tol, _ = attention(c)
    assert np.all(np.abs(out.download().reshape(n, d) - want) <= tol)
    for x in bufs + [ws]:
        x.free()
    cache.free()


# ------------------------------------------------------------------ appending


@pytest.mark.parametrize("n_pos,rot,theta", [(1, 2, 10000.0), (300, 64, 10000.0), (7, 48, 500000.0)])
def test_rotary_table(ctx, n_pos, rot, theta):
    """Each value is the nearest 32-bit number to cos or sin, give or take the 64-bit angle's own error."""
    from aurora_amd.gpu import GpuBuffer, RotaryTableKernel

    t = GpuBuffer.empty(ctx, n_pos * rot)
    RotaryTableKernel.new().dispatch_into(ctx, t, n_pos, rot, theta)
    got = t.download().reshape(n_pos, rot // 2, 2)
    a = np.arange(n_pos)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / rot)
    assert np.abs(got - np.stack([np.cos(a), np.sin(a)], -1)).max() <= U32 / 2 * 1.01  # |values| ≤ 1: half a step of 2^-24
    t.free()


def test_rotary_table_far_positions(ctx):
    """Position 2^22 − 1: a 32-bit angle would be off by 0.1."""
    from aurora_amd.gpu import GpuBuffer, RotaryTableKernel

    n, rot = 2**22, 8
    t = GpuBuffer.empty(ctx, n * rot)
    RotaryTableKernel.new().dispatch_into(ctx, t, n, rot)
    got = t.download().reshape(n, rot // 2, 2)[-1000:]
    a = np.arange(n - 1000, n)[:, None] * 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    assert np.abs(got - np.stack([np.cos(a), np.sin(a)], -1)).max() <= U32 / 2 * 1.01
    t.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,past,prefix,page,kv,group,dh,rot,pairs", [
    ([1], [0], 0, 1, 1, 1, 8, 8, False),
    ([1] * 5, [0, 15, 16, 3, 200], 33, 16, 2, 2, 32, 32, False),
    ([1] * 5, [0, 15, 16, 3, 200], 33, 16, 2, 2, 32, 32, True),
    ([40, 0, 7, 129], [0, 5, 100, 1], 500, 8, 3, 1, 48, 16, True),
    ([40, 0, 7, 129], [0, 5, 100, 1], 500, 8, 3, 1, 48, 16, False),
    ([3, 20], [4, 0], 0, 64, 2, 3, 64, 0, False),
    ([70], [30], 10, 32, 16, 1, 128, 64, False),
    ([2, 9], [1, 2], 5, 4, 1, 7, 72, 72, True),
])
def test_append_matches_float64(ctx, dtype, n, past, prefix, page, kv, group, dh, rot, pairs):
    """Rotated values lie within the roundings of a turn (two products, a sum, a table value of
    2^-25), copied columns and V are the inputs bit for bit (bf16: the nearest value), and every
    other row of the pools, and rows behind the last sequence, are as they were."""
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel, RotaryTableKernel

    rng = np.random.default_rng(sum(n) + dh + rot)
    c = Case(rng, n, [x + y for x, y in zip(n, past)], prefix, page, kv, group, dh, dtype, behind=3)
    dev = Device(ctx, c)
    before = [x.download() for x in (dev.k, dev.v)]
    row, d, n_pos = kv * dh, c.h * dh, prefix + c.max_own
    kx, vx = rng.standard_normal((2, c.n_tok, row + 4)).astype(np.float32)
    bk, bv = GpuBuffer.from_slice(ctx, kx.ravel()), GpuBuffer.from_slice(ctx, vx.ravel())
    table = GpuBuffer.empty(ctx, max(1, n_pos * rot))
    if rot:
        RotaryTableKernel.new().dispatch_into(ctx, table, n_pos, rot)
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, dev.q, d, bk, bv, row + 4, dev.out, d,
                                            table if rot else 0, n_pos, rot, c.h, pairs=pairs)
    got_q = dev.out.download().reshape(c.n_tok, d)
    got = [x.download() for x in (dev.k, dev.v)]
    at, pos = [], []
    for s in range(c.b):
        j = np.arange(c.length[s] - c.n[s], c.length[s])
        at += list(c.rows(c.pages[s], c.length[s])[j])
        pos += list(prefix + j)
    m = len(at)
    assert np.all(got_q[m:] == 7.5)

    def near(have, x, heads, bf16=False):
        want = rotate(x, pos, heads, dh, rot, pairs)
        size = np.abs(rotate(np.abs(x), pos, heads, dh, 0, pairs)).reshape(m, heads, dh)
        both = size.copy()
        if rot:  # |x| + |y| of each pair
            i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
            both[..., i0] = both[..., i1] = size[..., i0] + size[..., i1]
        tol = 3 * U32 * both.reshape(m, -1)
        if bf16:
            tol = tol * 1.01 + 2.0**-8 * (np.abs(want) + tol)
        assert np.all(np.abs(have - want) <= tol), float((np.abs(have - want) / tol).max())
        still = np.zeros(dh, bool)
        still[rot:] = True
        still = np.tile(still, heads)
        exact = from_bf16_bits(to_bf16_bits(x)) if bf16 else x
        assert np.array_equal(have[:, still], exact[:, still])

    near(got_q[:m], c.q[:m], c.h)
    value = (lambda x: from_bf16_bits(x)) if dtype == "bf16" else (lambda x: x)
    k, v = (value(x).reshape(-1, row) for x in got)
    near(k[at], kx[:m, :row], kv, dtype == "bf16")
    assert np.array_equal(v[at], from_bf16_bits(to_bf16_bits(vx[:m, :row])) if dtype == "bf16" else vx[:m, :row])
    other = np.ones(len(k), bool)
    other[at] = False
    for x, y in zip(got, before):
        x, y = (z.reshape(-1, row).view(np.uint16) for z in (x, y))
        assert np.array_equal(x[other], y[other])
    # in place, and without q
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, dev.q, d, bk, bv, row + 4, dev.q, d,
                                            table if rot else 0, n_pos, rot, c.h, pairs=pairs)
    assert np.array_equal(dev.q.download().reshape(c.n_tok, d)[:m], got_q[:m])
    dev.k.upload(before[0])
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, bk, bv, row + 4, 0, 0,
                                            table if rot else 0, n_pos, rot, 0, pairs=pairs)
    assert np.array_equal(dev.k.download().view(np.uint16), got[0].view(np.uint16))
    for x in (bk, bv, table):
        x.free()
    dev.free()


def test_append_drops_rows_without_a_page(ctx):
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel

    rng = np.random.default_rng(12)
    c = Case(rng, [1, 1, 3], [17, 20, 2], 0, 16, 1, 1, 32)
    c.pages[0, 1], c.pages[1, 1] = -1, c.n_pages
    dev = Device(ctx, c)
    before = [x.download() for x in (dev.k, dev.v)]
    x = rng.standard_normal((c.n_tok, 32)).astype(np.float32)
    b = GpuBuffer.from_slice(ctx, x.ravel())
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, dev.q, 32, b, b, 32, dev.out, 32, 0, 0, 0, 1)
    k = dev.k.download().reshape(-1, 32)
    at = c.rows(c.pages[2], 2)
    assert np.array_equal(k[at], x[3:5])  # the third sequence's two last tokens; its first has no place
    k[at] = before[0].reshape(-1, 32)[at]
    assert np.array_equal(k.view(np.uint32), before[0].reshape(-1, 32).view(np.uint32))
    out = dev.out.download().reshape(-1, 32)
    assert np.array_equal(out[[0, 1, 3, 4]], c.q[[0, 1, 3, 4]]) and np.all(out[2] == 7.5)
    b.free()
    dev.free()


@pytest.mark.parametrize("change,what", [
    (dict(rot_dim=12), "rot_dim"), (dict(rot_dim=72), "rot_dim"), (dict(n_pos=40), "table"), (dict(table=0), "table"),
    (dict(q_out=0), "together"), (dict(n_head=3), "n_head"), (dict(n_head=0), "n_head"), (dict(k=0), "k and v"),
    (dict(ld_kv=60), "ld_kv"), (dict(ld_kv=130), "ld_kv"), (dict(ld_q=64), "ld_q"), (dict(v="odd"), "16-byte"),
])
def test_append_refusals(ctx, change, what):
    from aurora_amd._lib import AuroraError

    c = Case(np.random.default_rng(13), [1, 1], [17, 20], 30, 16, 2, 1, 64)
    dev = Device(ctx, c)
    buf = dev.q.ptr
    args = dict(q=buf, ld_q=128, k=buf, v=buf, ld_kv=128, q_out=dev.out.ptr, ld_qo=128, table=dev.ws.ptr, n_pos=50,
                rot_dim=64, n_head=2, pairs=0)
    args.update({k: buf + 4 if v == "odd" else v for k, v in change.items()})
    with pytest.raises(AuroraError, match=what):
        ctx.call("aur_kv_append_paged", dev.cache.ref, dev.batch.ref, *args.values())
    dev.free()


@pytest.mark.parametrize("change,what", [
    (dict(q=0), "q and out"), (dict(out="odd"), "16-byte"), (dict(ld_q=124), "ld_q"), (dict(ld_o=130), "ld_o"),
    (dict(scratch=0), "scratch"), (dict(scratch_bytes="short"), "scratch"), (dict(n_head=3), "n_head"),
    (dict(n_head=0), "n_head"),
])
def test_attention_refusals(ctx, change, what):
    from aurora_amd._lib import AuroraError

    c = Case(np.random.default_rng(13), [1, 1], [17, 20], 3000, 16, 2, 1, 64)
    dev = Device(ctx, c)
    assert dev.ws_len > 0
    args = dict(q=dev.q.ptr, ld_q=128, out=dev.out.ptr, ld_o=128, lse=dev.lse.ptr, scratch=dev.ws.ptr,
                scratch_bytes=4 * dev.ws_len, n_head=2)
    args.update({k: dev.out.ptr + 4 if v == "odd" else 4 * dev.ws_len - 1 if v == "short" else v
                 for k, v in change.items()})
    with pytest.raises(AuroraError, match=what):
        ctx.call("aur_mha_paged", dev.cache.ref, dev.batch.ref, *args.values())
    assert np.all(dev.out.download() == 7.5)  # nothing ran
    dev.free()


def test_empty_batches(ctx):
    """No sequences, or no tokens: nothing to do, and no array is needed."""
    from aurora_amd.gpu import PagedBatch, PagedKvAppendKernel, PagedMhaKernel

    c = Case(np.random.default_rng(14), [1], [5])
    dev = Device(ctx, c)
    for batch in (PagedBatch(0, 0, 0, 0, 0, 4, 1, 0), PagedBatch(dev.off, dev.len, dev.pages, 1, 1, 0, 0, 16)):
        assert PagedMhaKernel.scratch_len(dev.cache, batch, 2) == 0
        PagedMhaKernel.new().dispatch_into(ctx, dev.cache, batch, dev.q.ptr, 64, dev.out.ptr, 64, 0, 0, 0, 2)
        PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, batch, 0, 0, 0, 0, 64, 0, 0, 0, 0, 0, 2)
    assert np.all(dev.out.download() == 7.5)
    dev.free()


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype,pairs,group", [("f32", False, 1), ("bf16", False, 2), ("f32", True, 3)])
def test_prefix_prompts_and_steps_together(ctx, dtype, pairs, group):
    """As a server uses them: the shared prefix is written once and attends to itself, prompts of
    different lengths follow it, then steps of one token; every row equals plain causal attention over
    its whole sequence, rotated by absolute positions, in float64."""
    from aurora_amd.gpu import (GpuBuffer, PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedMhaKernel,
                                RotaryTableKernel)

    rng = np.random.default_rng(15)
    kv, dh, rot, page, P, prompt, steps = 2, 64, 48, 16, 75, [9, 1, 33, 20], 3
    h, row, b = kv * group, kv * dh, len(prompt)
    own = max(prompt) + steps
    m = -(-own // page)
    first = -(-P // page)
    order = rng.permutation(first + b * m).astype(np.int32)
    cache = PagedKvCache.zeros(ctx, len(order), page, kv, dh, dtype)
    up = lambda x: GpuBuffer.from_slice(ctx, np.ascontiguousarray(x))  # noqa: E731
    prefix_pages, pages = up(order[:first]), up(order[first:])
    table = GpuBuffer.empty(ctx, (P + own) * rot)
    RotaryTableKernel.new().dispatch_into(ctx, table, P + own, rot)
    made = [prefix_pages, pages, table]
    data = [rng.standard_normal((3, P, h * dh)).astype(np.float32)]  # q, k, v of the prefix, then of each sequence
    data += [rng.standard_normal((3, n + steps, h * dh)).astype(np.float32) for n in prompt]
    out = [np.zeros((x.shape[1], h * dh)) for x in data]

    def call(parts, lens, past, tables, width, prefix_args, shared):
        """One append and one attention for `parts`: (which data, from, to) of each sequence."""
        n = [hi - lo for _, lo, hi in parts]
        rows = [np.concatenate([data[i][x, lo:hi] for i, lo, hi in parts]) for x in range(3)]
        q, k, v = up(rows[0].ravel()), up(rows[1][:, :row].ravel()), up(rows[2][:, :row].ravel())
        off, length = up(np.cumsum([0] + n).astype(np.int32)), up(np.array(lens, np.int32))
        res, total = GpuBuffer.empty(ctx, sum(n) * h * dh), sum(n)
        batch = PagedBatch(off, length, tables, len(n), width, total, max(n), max(lens), *prefix_args)
        PagedKvAppendKernel.new().dispatch_into(ctx, cache, batch, q, h * dh, k, v, row, q, h * dh, table, P + own, rot,
                                                h, pairs=pairs)
        ws_len = PagedMhaKernel.scratch_len(cache, batch, h)
        ws = GpuBuffer.empty(ctx, max(1, ws_len))
        PagedMhaKernel.new().dispatch_into(ctx, cache, batch, q, h * dh, res, h * dh, 0, ws, ws_len, h)
        got, at = res.download().reshape(total, -1), 0
        for (i, lo, hi), cnt in zip(parts, n):
            out[i][lo:hi] = got[at:at + cnt]
            at += cnt
        for x in (q, k, v, off, length, res, ws):
            x.free()

    call([(0, 0, P)], [P], 0, prefix_pages, first, (), False)
    shared = (prefix_pages, first, P)
    call([(i + 1, 0, n) for i, n in enumerate(prompt)], prompt, 0, pages, m, shared, True)
    for s in range(steps):
        call([(i + 1, n + s, n + s + 1) for i, n in enumerate(prompt)], [n + s + 1 for n in prompt], 0, pages, m, shared,
             True)

    store = (lambda x: from_bf16_bits(to_bf16_bits(x.astype(np.float32))).astype(np.float64)) if dtype == "bf16" \
        else (lambda x: x)
    for i in range(1, b + 1):
        x = np.concatenate([data[0], data[i]], 1)
        pos = np.arange(x.shape[1])
        q = rotate(x[0], pos, h, dh, rot, pairs)
        k = store(rotate(x[1][:, :row], pos, kv, dh, rot, pairs))
        v = store(x[2][:, :row].astype(np.float64))
        k, v = (np.repeat(y.reshape(-1, kv, dh), group, 1) for y in (k, v))
        want, _ = causal_attention_f64(q.reshape(1, -1, h, dh), k[None], v[None])
        got = np.concatenate([out[0], out[i]])
        # 32 bits: scores of 64 products within (dh + 6)·2^-24·Σ|q||k|/8 ≤ 70·2^-24·64·9/8 (values to 3), twice;
        # bf16: a key whose 64-bit value lies at a rounding's border may round the other way, a step of 2^-7
        # of one column of one key: scores move by 2^-7·9/8, which is rare and leaves its mark on few rows
        tol = 6e-4 if dtype == "f32" else 2e-2
        err = np.abs(got - want.reshape(len(got), -1)).max()
        assert err <= tol, err
    for x in made:
        x.free()
    cache.free()
