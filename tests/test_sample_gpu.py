"""Choosing the next token on the GPU against the definition in float64 (tests/e4m3_ref.py: sample), and against
whole numbers where borders are met exactly."""
import numpy as np
import pytest

from tests.e4m3_ref import sample, sample_exact

pytestmark = pytest.mark.gpu


def _run(ctx, x, u, temperature=None, top_k=None, top_p=None, min_p=None, ld=None, offset=0, logprob=True):
    """(tokens, logprob) for rows x [b, vocab] in a buffer of row stride ld, `offset` floats from its start."""
    from aurora_amd.gpu import GpuBuffer, SampleKernel

    b, vocab = x.shape
    ld = ld or vocab
    held = np.full(offset + b * ld, 1e30, np.float32)  # what lies between the rows is larger than all of them
    np.lib.stride_tricks.as_strided(held[offset:], (b, vocab), (4 * ld, 4))[:] = x
    bufs = [GpuBuffer.from_slice(ctx, held)]
    put = lambda v, t: 0 if v is None else bufs.append(GpuBuffer.from_slice(ctx, np.broadcast_to(np.asarray(v, t), (b,)))) or bufs[-1]  # noqa: E731
    u, t, k, p, m = put(u, np.float32), put(temperature, np.float32), put(top_k, np.int32), put(top_p, np.float32), put(min_p, np.float32)
    tokens = GpuBuffer.from_slice(ctx, np.full(b + 1, -5, np.int32))
    lp = GpuBuffer.from_slice(ctx, np.full(b + 1, 7.5, np.float32))
    logits = bufs[0].ptr + 4 * offset if offset else bufs[0]
    SampleKernel.new().dispatch_into(ctx, logits, ld, u, tokens, lp if logprob else 0, b, vocab, t, k, p, m)
    got = tokens.download(), lp.download()
    for buf in bufs + [tokens, lp]:
        buf.free()
    assert got[0][b] == -5 and got[1][b] == 7.5
    return got[0][:b], got[1][:b]


def _check(x, u, tokens, logprob, **kw):
    b = len(x)
    near_border = 0
    for r in range(b):
        args = {n: (np.broadcast_to(np.asarray(v, np.int32 if n == "top_k" else np.float32), (b,))[r]) for n, v in kw.items()
                if v is not None}
        with np.errstate(all="ignore"):
            token, lp, near = sample(x[r], np.float32(u[r]), **{n: float(v) if n != "top_k" else int(v) for n, v in args.items()})
        if tokens[r] != token:  # so near a border, sums in another order may fall on its other side
            assert near < 1e-9, (r, tokens[r], token, near)
            near_border += 1
            continue
        if np.isfinite(lp):
            # float64 throughout, weights in units of 2^-43 at least; then one rounding to 32 bits
            assert abs(logprob[r] - lp) <= 2.0**-24 * abs(lp) + 1e-9, (r, logprob[r], lp)
        else:
            assert logprob[r] == lp
    assert near_border <= b // 10


VOCABS = [1, 2, 3, 63, 64, 65, 255, 256, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8192, 8191, 16385, 32768, 65536, 70001, 131072]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("top_k,top_p,min_p", [(None, None, None), (50, None, None), (None, 0.9, None), (None, None, 0.05),
                                               (40, 0.95, 0.02), (0, 1.0, 0.0), (700, 0.5, None)])
def test_matches_the_definition(ctx, vocab, top_k, top_p, min_p):
    rng = np.random.default_rng(vocab)
    b = 5
    x = (2.5 * rng.standard_normal((b, vocab))).astype(np.float32)
    u, t = rng.random(b).astype(np.float32), rng.uniform(0.5, 1.5, b).astype(np.float32)
    kw = dict(temperature=t, top_k=top_k, top_p=top_p, min_p=min_p)
    tokens, lp = _run(ctx, x, u, ld=vocab + vocab % 3, **kw)
    _check(x, u, tokens, lp, **kw)


@pytest.mark.parametrize("vocab", [300, 5000, 20000, 50000])
def test_every_row_has_its_own_filters(ctx, vocab):
    rng = np.random.default_rng(1)
    b = 64
    x = (3 * rng.standard_normal((b, vocab))).astype(np.float32)
    u = rng.random(b).astype(np.float32)
    kw = dict(temperature=rng.choice([0.0, 0.3, 1.0, 2.0, -1.0, np.nan], b), top_k=rng.choice([-1, 0, 1, 2, 100, 5000, 9999, 60000], b),
              top_p=rng.choice([0.0, 0.1, 0.9, 1.0, 1.5, np.nan], b), min_p=rng.choice([-1.0, 0.0, 0.1, 1.0, 3.0, np.nan], b))
    tokens, lp = _run(ctx, x, u, **kw)
    _check(x, u, tokens, lp, **kw)


@pytest.mark.parametrize("vocab", [7, 900, 3000, 9000, 40001])
def test_rows_that_are_not_16_byte_aligned(ctx, vocab):
    rng = np.random.default_rng(2)
    x = (2 * rng.standard_normal((4, vocab))).astype(np.float32)
    u = rng.random(4).astype(np.float32)
    kw = dict(top_k=min(20, vocab), top_p=0.9)
    want = _run(ctx, x, u, **kw)
    for offset, ld in ((1, vocab), (2, vocab + 1), (3, vocab + 5), (0, -(-vocab // 4) * 4), (1, -(-vocab // 4) * 4)):
        got = _run(ctx, x, u, ld=ld, offset=offset, **kw)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    _check(x, u, *want, **kw)


@pytest.mark.parametrize("vocab", [64, 1500, 6000])
def test_frequencies_follow_the_shares(ctx, vocab):
    """Evenly spaced random numbers give every token its share of them, but for one."""
    rng = np.random.default_rng(3)
    n = 2000
    x = np.tile((2 * rng.standard_normal(vocab)).astype(np.float32), (n, 1))
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens, _ = _run(ctx, x, u)
    p = np.exp(x[0].astype(np.float64) - x[0].max())
    count = np.bincount(tokens, minlength=vocab)
    assert np.all(np.abs(count - n * p / p.sum()) <= 1.01) and np.all(np.diff(tokens) >= 0)


def _exact(ctx, x, weights, u, top_k=0, top_p=1.0):
    tokens, lp = _run(ctx, x, u, top_k=top_k, top_p=top_p)
    for r in range(len(x)):
        order = np.argsort(-x[r], kind="stable")
        want = sample_exact([int(w) for w in weights[r]], order.tolist(), top_k, float(np.float32(top_p)), float(np.float32(u[r])))
        assert tokens[r] == want, (r, tokens[r], want)
    return lp


@pytest.mark.parametrize("vocab", [1, 5, 256, 1024, 3000, 20000, 33000])
@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (0, 0.5), (0, 0.25), (37, 1.0), (37, 0.5), (2048, 0.75)])
def test_equal_logits_go_by_index(ctx, vocab, top_k, top_p):
    """One value throughout, where every border is met exactly and the lowest indexes are kept."""
    b = 6
    x = np.full((b, vocab), -3.25, np.float32)
    lp = _exact(ctx, x, np.ones((b, vocab), int), [0.0, 0.125, 0.5, 0.75, 1 - 2.0**-24, 0.3], top_k if top_k < vocab else 0, top_p)
    kept = min(top_k or vocab, vocab)
    kept = -int(-kept * top_p // 1) if top_p < 1 else kept
    np.testing.assert_allclose(lp, -np.log(kept), rtol=1e-6, atol=1e-7)


def test_ties_at_the_borders(ctx):
    """Values of ln 2 apart in many copies each: weights of powers of two."""
    rng = np.random.default_rng(4)
    b, vocab = 8, 6000
    e = rng.integers(0, 4, (b, vocab))
    x = np.array([0.0, -100.0, -200.0, -300.0], np.float32)[e]  # weights 1 and (far below a unit) 0
    w = np.array([1, 0, 0, 0])[e]
    for k, p in ((0, 0.5), (100, 1.0), (1000, 0.125), (1600, 1.0), (0, 1.0)):
        _exact(ctx, x, w, rng.integers(0, 64, b) / 64, k, p)


@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (1500, 1.0), (0, 0.5), (2500, 0.9), (3, 1.0)])
@pytest.mark.parametrize("what", ["band", "outlier", "subnormal", "far apart", "two bands"])
@pytest.mark.parametrize("vocab", [5000, 40000])
def test_logits_that_crowd_one_range(ctx, vocab, what, top_k, top_p):
    rng = np.random.default_rng(5)
    b = 4
    x = rng.permuted(np.tile(np.arange(vocab), (b, 1)), axis=1).astype(np.float64)
    if what == "band":
        x = 1 + x * 2.0**-23
    elif what == "outlier":
        x = np.where(x == 17, -3e38, x * 1e-3)
    elif what == "subnormal":
        x = x * 2.0**-149
    elif what == "far apart":
        x = np.where(x < 2500, x * 1e-4, -3.4e38 + x * 1e33)
    else:
        x = np.where(x < 2500, 5 + x * 2.0**-20, -5 + x * 2.0**-20)
    x = x.astype(np.float32)
    u = rng.random(b).astype(np.float32)
    if what == "subnormal":  # all weights are 1, and borders are met exactly
        _exact(ctx, x, np.ones((b, vocab), int), u, top_k, top_p)
        return
    kw = dict(top_k=top_k, top_p=top_p)
    tokens, lp = _run(ctx, x, u, **kw)
    _check(x, u, tokens, lp, **kw)


@pytest.mark.parametrize("vocab", [4, 900, 2000, 5000, 34000])
@pytest.mark.parametrize("kw", [{}, dict(top_k=3), dict(top_p=0.5), dict(top_k=1500, top_p=0.7, min_p=0.1), dict(temperature=0.0)])
def test_infinities_and_nan(ctx, vocab, kw):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, 1:] = -np.inf
    x[3, vocab // 2] = np.inf
    x[4, ::2] = np.inf
    x[4, 1::2] = np.nan
    x[5, rng.random(vocab) < 0.5] = np.nan
    x[5, vocab - 1] = 9.0
    u = np.array([0.5, 0.5, 0.99, 0.7, 0.3, 0.2], np.float32)
    tokens, lp = _run(ctx, x, u, **kw)
    assert tokens[0] == 0 and tokens[1] == 0 and np.isneginf(lp[:2]).all()
    _check(x[2:], u[2:], tokens[2:], lp[2:], **kw)


@pytest.mark.parametrize("vocab", [3000, 36000])
def test_temperatures_and_numbers_at_the_ends(ctx, vocab):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((8, vocab)).astype(np.float32)
    t = np.array([1e-45, 1e-30, 1e30, 3.4e38, np.inf, 0.01, 100.0, 1.0], np.float32)
    u = np.full(8, 0.6, np.float32)
    tokens, lp = _run(ctx, x, u, temperature=t)
    _check(x, u, tokens, lp, temperature=t)
    u = np.array([0.0, -1.0, np.nan, 1.0, 2.0, np.inf, -np.inf, 2.0**-149], np.float32)
    tokens, _ = _run(ctx, x, u, top_k=20)
    for r in range(8):
        kept = np.sort(np.argsort(-x[r], kind="stable")[:20])
        assert tokens[r] == (kept[-1] if u[r] >= 1 else kept[0])
    kw = dict(temperature=t, top_k=500, top_p=0.7, min_p=0.2)
    u = np.full(8, 0.6, np.float32)
    tokens, lp = _run(ctx, x, u, **kw)
    _check(x, u, tokens, lp, **kw)


@pytest.mark.parametrize("vocab", [33000, 49152, 131072, 200003])
@pytest.mark.parametrize("kw", [{}, dict(min_p=0.3), dict(min_p=1e-4), dict(top_k=30000), dict(top_k=3), dict(top_k=20000, top_p=0.999),
                                dict(top_p=0.01), dict(top_p=0.9999), dict(top_k=2000, top_p=0.999, min_p=0.001),
                                dict(top_p=0.99, min_p=0.4), dict(top_k=500, min_p=0.0001)])
def test_rows_that_several_blocks_share(ctx, vocab, kw):
    rng = np.random.default_rng(vocab)
    b = 9
    x = (rng.choice([0.5, 2.5, 8.0], (b, 1)) * rng.standard_normal((b, vocab))).astype(np.float32)
    x[1] = np.round(x[1] * 8) / 8  # equal logits in all segments
    x[2, :20000] = -np.inf
    x[3] = np.sort(x[3])
    u = rng.random(b).astype(np.float32)
    tokens, lp = _run(ctx, x, u, **kw)
    _check(x, u, tokens, lp, **kw)


def test_captured_into_a_graph(ctx):
    """A call of each size captured once and replayed with new logits and numbers: as an eager call."""
    import ctypes

    from aurora_amd._lib import load
    from aurora_amd.gpu import GpuBuffer, SampleKernel
    from tests.test_paged_gpu import _hip

    hip, stream = _hip(), load().aur_stream(ctx.ptr)
    rng = np.random.default_rng(9)
    for vocab in (200, 6000, 40000):
        b = 5
        logits, u = GpuBuffer.zeros(ctx, b * vocab), GpuBuffer.zeros(ctx, b)
        t, p = GpuBuffer.from_slice(ctx, np.full(b, 0.8, np.float32)), GpuBuffer.from_slice(ctx, np.full(b, 0.9, np.float32))
        out = [(GpuBuffer.zeros(ctx, b, np.int32), GpuBuffer.zeros(ctx, b)) for _ in range(2)]
        kernels = SampleKernel.new(), SampleKernel.new()
        for kernel in kernels:
            kernel.reserve(ctx, b, vocab)
        call = lambda i: kernels[i].dispatch_into(ctx, logits, vocab, u, *out[i], b, vocab, t, 0, p, 0)  # noqa: E731
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        ctx.sync()
        assert hip.hipStreamBeginCapture(stream, 1) == 0  # hipStreamCaptureModeThreadLocal
        try:
            call(0)
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for _ in range(4):
            x, r = (3 * rng.standard_normal((b, vocab))).astype(np.float32), rng.random(b).astype(np.float32)
            logits.upload(x.ravel()), u.upload(r)
            assert hip.hipGraphLaunch(exe, stream) == 0
            ctx.sync()
            call(1)
            for got, want in zip(*out):
                assert np.array_equal(got.download(), want.download())
            _check(x, r, out[0][0].download(), out[0][1].download(), temperature=0.8, top_p=0.9)
        hip.hipGraphExecDestroy(exe), hip.hipGraphDestroy(graph)
        for z in (logits, u, t, p, *out[0], *out[1], *kernels):
            z.free()


def test_without_logprob_and_twice_the_same(ctx):
    rng = np.random.default_rng(8)
    x = (2 * rng.standard_normal((300, 2500))).astype(np.float32)
    u = rng.random(300).astype(np.float32)
    kw = dict(top_k=1200, top_p=0.8)
    a, lp = _run(ctx, x, u, **kw)
    b, other = _run(ctx, x, u, logprob=False, **kw)
    assert np.array_equal(a, b) and np.all(other == 7.5)
    c, lp2 = _run(ctx, x, u, **kw)
    assert np.array_equal(a, c) and np.array_equal(lp, lp2)
