"""Calls of the 8-bit cache's kernels and of choosing tokens that their documentation allows or refuses, next to
those of tests/test_e4m3_gpu.py and tests/test_sample_gpu.py."""
import numpy as np
import pytest

from tests.e4m3_ref import NUMBERS, Case8, sample
from tests.paged_ref import Case, attention
from tests.paged_tiles import attention_blocks
from tests.test_e4m3_gpu import Device8, _append
from tests.test_paged_gpu import Device

pytestmark = pytest.mark.gpu


def test_two_contexts_at_once_and_the_same_bits(ctx):
    """Calls on two streams with a scratch each, and a call again, give the same bits."""
    from aurora_amd.gpu import GpuContext

    for n, group in (([1] * 20, 1), ([30, 1, 9], 2)):
        c = Case8(np.random.default_rng(10), n, [x + 10 * i for i, x in enumerate(n)], 2000, 64, 4, group, 64, 16)
        dev = Device8(ctx, c)
        dev.attend()
        first = dev.result()
        with GpuContext.new(0) as other:
            dev2 = Device8(other, c)
            other.sync()
            for _ in range(5):
                dev.attend()
                dev2.attend()
            for got in (dev.result(), dev2.result()):
                for x, y in zip(first, got):
                    assert np.array_equal(x, y)
            dev2.free()
        dev.free()


def test_choices_of_two_contexts_at_once(ctx):
    """Two objects on two streams; an object that goes from one context to the other takes a scratch there."""
    from aurora_amd.gpu import GpuBuffer, GpuContext, SampleKernel

    rng = np.random.default_rng(3)
    b, vocab = 12, 50000
    x = [(3 * rng.standard_normal((b, vocab))).astype(np.float32) for _ in range(2)]
    u = rng.random(b).astype(np.float32)
    p = np.full(b, 0.9, np.float32)

    def buffers(on, rows):
        return [GpuBuffer.from_slice(on, rows.ravel()), GpuBuffer.from_slice(on, u), GpuBuffer.zeros(on, b, np.int32),
                GpuBuffer.zeros(on, b), GpuBuffer.from_slice(on, p)]

    def call(kernel, on, bufs):
        kernel.dispatch_into(on, bufs[0], vocab, bufs[1], bufs[2], bufs[3], b, vocab, 0, 0, bufs[4])

    with GpuContext.new(0) as other:
        kernels, bufs = [SampleKernel.new(), SampleKernel.new()], [buffers(ctx, x[0]), buffers(other, x[1])]
        ctx.sync(), other.sync()
        for _ in range(5):
            call(kernels[0], ctx, bufs[0]), call(kernels[1], other, bufs[1])
        got = [z[2].download() for z in bufs]
        for rows, tokens in zip(x, got):
            for r in range(b):
                token, _, near = sample(rows[r], u[r], top_p=float(p[r]))
                assert tokens[r] == token or near < 1e-9
        call(kernels[0], other, bufs[1])
        assert np.array_equal(bufs[1][2].download(), got[1])
        for z in bufs[0] + bufs[1]:
            z.free()
        for k in kernels:
            k.free()


def test_a_captured_choice_outlives_a_larger_call(ctx):
    """An object whose call was captured, then used for more rows: the graph still has its scratch."""
    import ctypes

    from aurora_amd._lib import load
    from aurora_amd.gpu import GpuBuffer, SampleKernel
    from tests.test_paged_gpu import _hip

    hip, stream = _hip(), load().aur_stream(ctx.ptr)
    rng = np.random.default_rng(4)
    vocab, kernel = 40000, SampleKernel.new()
    sets = {}
    for b in (2, 30):
        x = (3 * rng.standard_normal((b, vocab))).astype(np.float32)
        sets[b] = [GpuBuffer.from_slice(ctx, x.ravel()), GpuBuffer.from_slice(ctx, rng.random(b).astype(np.float32)),
                   GpuBuffer.zeros(ctx, b, np.int32), GpuBuffer.from_slice(ctx, np.full(b, 0.8, np.float32))]
    call = lambda b: kernel.dispatch_into(ctx, sets[b][0], vocab, sets[b][1], sets[b][2], 0, b, vocab, 0, 0, sets[b][3])  # noqa: E731
    call(2)
    want = sets[2][2].download()
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(stream, 1) == 0  # hipStreamCaptureModeThreadLocal
    try:
        call(2)
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
    call(30)
    large = sets[30][2].download()
    for _ in range(3):
        sets[2][2].upload(np.full(2, -1, np.int32))
        assert hip.hipGraphLaunch(exe, stream) == 0
        ctx.sync()
        assert np.array_equal(sets[2][2].download(), want)
        call(30)
        assert np.array_equal(sets[30][2].download(), large)
    hip.hipGraphExecDestroy(exe), hip.hipGraphDestroy(graph)
    for b in sets:
        for z in sets[b]:
            z.free()
    kernel.free()


@pytest.mark.parametrize("n,group", [(300, 1), (1, 1), (1, 16), (3, 4)])
def test_pool_beyond_32_bit_offsets(ctx, n, group):
    """Pages whose elements start beyond 2^32 bytes: appended to, attended to and read back."""
    from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedKvReadKernel, PagedMhaKernel

    kv, dh, page, own, block = 16, 128, 256, 300, 32
    row, d = kv * dh, kv * dh * group
    n_pages = (2**32 + 2**28) // (page * row)
    rng = np.random.default_rng(16)
    c = Case8(rng, [n], [own], 0, page, kv, group, dh, block)
    new = lambda m: GpuBuffer.empty(ctx, m, np.uint8)  # noqa: E731
    scales = n_pages * kv * (page // block)
    cache = PagedKvCache(new(n_pages * page * row), new(n_pages * page * row), n_pages, page, kv, dh, "e4m3", new(scales),
                         new(scales), block)
    up = lambda x: GpuBuffer.from_slice(ctx, x)  # noqa: E731
    k, v = rng.standard_normal((2, own, row)).astype(np.float32)
    bufs = [up(np.array([0, own, 0, n], np.int32)), up(np.array([own], np.int32)),
            up(np.array([n_pages - 1, n_pages - 3], np.int32)), up(k.ravel()), up(v.ravel()), up(c.q.ravel()),
            GpuBuffer.empty(ctx, n * d), GpuBuffer.empty(ctx, own * row), GpuBuffer.empty(ctx, own * row)]
    off, length, pg, bk, bv, bq, out, ko, vo = bufs
    PagedKvAppendKernel.new().dispatch_into(ctx, cache, PagedBatch(off, length, pg, 1, 2, own, own, own), 0, 0, bk, bv,
                                            row, 0, 0, 0, 0, 0, kv)
    batch = PagedBatch(off.ptr + 8, length, pg, 1, 2, n, n, own)
    ws_len = PagedMhaKernel.scratch_len(cache, batch, c.h)
    ws = GpuBuffer.empty(ctx, max(1, ws_len))
    PagedMhaKernel.new().dispatch_into(ctx, cache, batch, bq, d, out, d, 0, ws, ws_len, c.h)
    PagedKvReadKernel.new().dispatch_into(ctx, cache, batch, ko, vo, row, 0, own)
    # the same bytes in a pool of two pages
    c.n, c.off = np.array([own]), np.array([0, own])
    c.pages, c.n_pages = np.array([[0, 1]], np.int32), 2
    c.kb, c.vb = (np.zeros((2 * page, row), np.uint8) for _ in range(2))
    c.ks, c.vs = (np.zeros((2, kv, page // block), np.uint8) for _ in range(2))
    c.append(k.reshape(own, kv, dh), v.reshape(own, kv, dh))
    assert np.array_equal(ko.download().reshape(own, row), c.kp[:own])
    assert np.array_equal(vo.download().reshape(own, row), c.vp[:own])
    c.n, c.off = np.array([n]), np.array([0, n])
    want, _, tol, _ = attention(c)
    assert np.all(np.abs(out.download().reshape(n, d) - want) <= tol)
    for x in bufs + [ws]:
        x.free()
    cache.free()


@pytest.mark.parametrize("n,prefix,group", [([1, 1, 1, 1], 100, 1), ([1] * 40, 2000, 1), ([9, 30, 2, 20], 100, 2),
                                            ([60, 70, 90, 80], 1500, 2)])
@pytest.mark.parametrize("block", [1, 16])
def test_values_beyond_the_bounds_touch_nothing_else(ctx, n, prefix, group, block):
    """Offsets and lengths that break the host's bounds, or are not ascending, are cut to them: other rows of the
    outputs, other pages' elements and scales stay as they were, and sound sequences keep their results."""
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel, PagedKvReadKernel

    rng = np.random.default_rng(21)
    c = Case8(rng, n, [x + 30 for x in n], prefix, 16, 2, group, 64, block, behind=5)
    dev = Device8(ctx, c, ld_q=c.h * 64 + 4, ld_o=c.h * 64 + 4)
    want, want_lse, tol, tol_lse = attention_blocks(c)
    x = GpuBuffer.from_slice(ctx, rng.standard_normal(c.n_tok * 128).astype(np.float32))
    held = dev.bytes()
    named = np.zeros(c.n_pages, bool)
    for s in range(c.b):
        named[c.pages[s, :-(-c.length[s] // 16)]] = True
    off, length = c.off.copy(), c.length.astype(np.int32)
    keys = prefix + c.max_own
    rows_out = GpuBuffer.zeros(ctx, c.b * keys * 128)
    for bad_off, bad_len in [({-1: c.n_tok + 1000}, {}), ({-1: 2**31 - 1}, {0: -5}), ({1: -2**31}, {1: 2**31 - 1}),
                             ({0: -7, -1: off[-2]}, {0: -2**31, 1: c.max_own + 1})]:
        o, l = off.copy(), length.copy()
        for i, v in bad_off.items():
            o[i] = v
        for i, v in bad_len.items():
            l[i] = v
        dev.off.upload(o), dev.len.upload(l)
        dev.out.upload(np.full(dev.out.len, 7.5, np.float32)), dev.lse.upload(np.full(dev.lse.len, 7.5, np.float32))
        dev.attend()
        out, lse = dev.result()
        assert np.all(out[:, c.h * 64:] == 7.5)
        whole = [s for s in range(c.b) if (o[s], o[s + 1], l[s]) == (off[s], off[s + 1], length[s])]
        assert whole
        for s in whole:
            rows = slice(off[s], off[s + 1])
            assert np.all(np.abs(out[rows, :c.h * 64] - want[rows]) <= tol[rows]), s
            assert np.all(np.abs(lse[rows] - want_lse[rows]) <= tol_lse[rows]), s
        last = min(max(int(o.max()), 0), c.n_tok)
        assert np.all(out[last:] == 7.5) and np.all(lse[last:] == 7.5)
        PagedKvReadKernel.new().dispatch_into(ctx, dev.cache, dev.batch, rows_out, 0, 128, 0, keys)
        got = rows_out.download().reshape(c.b, keys, 128)
        for s in range(c.b):
            cut = prefix + min(max(int(l[s]), 0), c.max_own)
            assert np.all(got[s, cut:] == 0)
            if l[s] == length[s]:
                assert np.array_equal(got[s, :cut], c.keys(s)[0].reshape(-1, 128).astype(np.float32))
        PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, x, x, 128, 0, 0, 0, 0, 0, 0)
        for have, was in zip(dev.bytes(), held):
            have, was = (y.reshape(c.n_pages, -1) for y in (have, was))
            assert np.array_equal(have[~named], was[~named])
        for buf, was in zip((dev.k, dev.v, dev.ks, dev.vs), held):
            buf.upload(was.ravel())
    x.free(), rows_out.free()
    dev.free()


def test_every_byte_at_every_scale(ctx):
    """Reading back: each of the 256 bytes at each of the 256 scales is the nearest 32-bit number to its value."""
    from aurora_amd.gpu import GpuBuffer, PagedKvReadKernel

    c = Case8(np.random.default_rng(1), [1], [512], 0, 512, 1, 1, 128, 1)
    c.pages = np.array([[0]], np.int32)
    token = np.arange(512)
    c.kb[:512] = (np.arange(128)[None] + 128 * (token[:, None] % 2)).astype(np.uint8)
    c.vb[:512] = c.kb[:512][:, ::-1]
    c.ks[0, 0], c.vs[0, 0] = token // 2, 255 - token // 2
    dev = Device8(ctx, c)
    outs = [GpuBuffer.zeros(ctx, 512 * 128) for _ in range(2)]
    PagedKvReadKernel.new().dispatch_into(ctx, dev.cache, dev.batch, *outs, 128, 0, 512)
    for out, byte, scale in zip(outs, (c.kb, c.vb), (c.ks, c.vs)):
        got, e = out.download().reshape(512, 128), scale[0, 0].astype(np.float64)[:, None]
        with np.errstate(over="ignore", invalid="ignore"):
            want = np.where(e == 255, np.nan, NUMBERS[byte[:512]] * 2.0 ** (e - 127)).astype(np.float32)
        assert np.array_equal(got, want, equal_nan=True)
        out.free()
    dev.free()


@pytest.mark.parametrize("n,prefix,group", [([1, 1, 1], 400, 1), ([1] * 40, 300, 1), ([90, 70], 60, 2), ([5, 6], 30, 4)])
@pytest.mark.parametrize("dh", [24, 64, 128])
@pytest.mark.parametrize("k_e,v_e", [((0,), (-60, 0, 9)), ((0, -70), (0,)), ((0, -117), (0, -117, 30)), ((-117,), (-117,))])
def test_scales_far_apart(ctx, n, prefix, group, dh, k_e, v_e):
    """Neighbouring blocks whose scales lie further apart than a half's range, the smallest ones among them."""
    rng = np.random.default_rng(dh + len(n))
    c = Case8(rng, n, [x + 20 for x in n], prefix, 16, 1, group, dh, 4)
    for s, e in ((c.ks, k_e), (c.vs, v_e)):
        s[...] = np.where(s == 255, 255, np.maximum(s + rng.choice(e, s.shape), 0 if min(e) > -117 else 10))
    with np.errstate(invalid="ignore"):
        c.refresh()
    dev = Device8(ctx, c)
    dev.attend()
    out, lse = dev.result()
    want, want_lse, tol, tol_lse = attention_blocks(c)
    rows = int(c.off[-1])
    # values of 2^-117·2^-9 and their sums are subnormal: 2^-149 for each of the roundings that such a sum has
    least = 2.0**-149 * (prefix + max(n) + 20) * (max(v_e) == -117)
    assert np.all(np.abs(out[:rows] - want[:rows]) <= tol[:rows] + least)
    assert np.all(np.abs(lse[:rows] - want_lse[:rows]) <= tol_lse[:rows])
    dev.free()


@pytest.mark.parametrize("n,prefix,group", [([1, 1, 1], 400, 1), ([1] * 40, 300, 1), ([90, 70], 60, 2), ([5, 6], 30, 4)])
@pytest.mark.parametrize("larger", [30, 26])
def test_the_smallest_scale_beside_small_ones(ctx, n, prefix, group, larger):
    """Values of the smallest scale beside ones 2^20 and 2^16 larger, which do not hide them."""
    rng = np.random.default_rng(len(n))
    c = Case8(rng, n, [x + 20 for x in n], prefix, 16, 1, group, 64, 4)
    c.vs[...] = np.where(c.vs == 255, 255, rng.choice([10, larger], c.vs.shape, p=[0.9, 0.1]))
    with np.errstate(invalid="ignore"):
        c.refresh()
    dev = Device8(ctx, c)
    dev.attend()
    out, _ = dev.result()
    want, _, tol, _ = attention_blocks(c)
    rows = int(c.off[-1])
    assert np.all(np.abs(out[:rows] - want[:rows]) <= tol[:rows] + 2.0**-149 * (prefix + max(n) + 20))
    dev.free()


@pytest.mark.parametrize("n,prefix,group", [([1, 1, 1], 400, 1), ([1] * 40, 300, 1), ([90, 70], 60, 2), ([5, 6], 30, 4)])
@pytest.mark.parametrize("apart", [15, 16, 21, 22, 23])
@pytest.mark.parametrize("of_k", [False, True])
def test_scales_at_the_border(ctx, n, prefix, group, apart, of_k):
    """Largest and smallest numbers of scales about as far apart as the halves' products take."""
    rng = np.random.default_rng(apart + len(n))
    c = Case8(rng, n, [x + 20 for x in n], prefix, 16, 1, group, 64, 2)
    byte, scale = (c.kb, c.ks) if of_k else (c.vb, c.vs)
    scale[...] = np.where(scale == 255, 255, 127 - 8 * of_k - apart * rng.integers(0, 2, scale.shape))
    ends = rng.choice(np.array([1, 126, 129, 254], np.uint8), byte.shape)  # ±2^-9, ±448
    byte[...] = np.where(rng.random(byte.shape) < 0.5, ends, byte)
    if of_k:  # scores of a few units for the larger ones
        c.q *= np.float32(2.0**-8)
    with np.errstate(invalid="ignore"):
        c.refresh()
    dev = Device8(ctx, c)
    dev.attend()
    out, lse = dev.result()
    want, want_lse, tol, tol_lse = attention_blocks(c)
    rows = int(c.off[-1])
    assert np.all(np.abs(out[:rows] - want[:rows]) <= tol[:rows])
    assert np.all(np.abs(lse[:rows] - want_lse[:rows]) <= tol_lse[:rows])
    dev.free()


@pytest.mark.parametrize("change,what", [
    (dict(ld=124), "ld=124"), (dict(ld=130), "ld=130"), (dict(k="odd"), "16-byte"), (dict(v="odd"), "16-byte"),
    (dict(count=51), "keys 0 to 51"), (dict(first=2**32 - 1, count=2), "keys"), (dict(first=51, count=0), "keys 51"),
])
def test_read_refusals(ctx, change, what):
    from aurora_amd._lib import AuroraError

    for case, device in ((Case8, Device8), (Case, Device)):
        c = case(np.random.default_rng(13), [1, 1], [17, 20], 30, 16, 2, 1, 64)
        dev = device(ctx, c)
        args = dict(k=dev.out.ptr, v=dev.out.ptr, ld=128, first=0, count=50)
        args.update({k: dev.out.ptr + 4 if v == "odd" else v for k, v in change.items()})
        with pytest.raises(AuroraError, match=what):
            ctx.call("aur_kv_read_paged", dev.cache.ref, dev.batch.ref, *args.values())
        assert np.all(dev.out.download() == 7.5)  # nothing ran
        dev.free()


@pytest.mark.parametrize("change,what", [
    (dict(vocab=0), "vocab=0"), (dict(ld=39999), "ld=39999"), (dict(logits=0), "null"), (dict(u=0), "null"),
    (dict(tokens=0), "null"), (dict(scratch=0), "scratch"), (dict(scratch="odd"), "scratch"), (dict(scratch_bytes="short"), "scratch"),
    (dict(vocab=2**20 + 1, ld=2**21), "vocab"), (dict(b=2**20), "b="), (dict(ld=2**31), "ld="),
])
def test_choice_refusals(ctx, change, what):
    from aurora_amd._lib import AuroraError
    from aurora_amd.gpu import GpuBuffer, SampleKernel

    b, vocab = 2, 40000
    need = SampleKernel.scratch_bytes(b, vocab)
    bufs = [GpuBuffer.zeros(ctx, b * vocab), GpuBuffer.zeros(ctx, b), GpuBuffer.from_slice(ctx, np.full(b, -5, np.int32)),
            GpuBuffer.empty(ctx, need, np.uint8)]
    args = dict(logits=bufs[0].ptr, ld=vocab, u=bufs[1].ptr, temperature=0, top_k=0, top_p=0, min_p=0, tokens=bufs[2].ptr,
                logprob=0, scratch=bufs[3].ptr, scratch_bytes=need, b=b, vocab=vocab)
    args.update({k: bufs[3].ptr + 8 if v == "odd" else need - 1 if v == "short" else v for k, v in change.items()})
    with pytest.raises(AuroraError, match=what):
        ctx.call("aur_sample", *args.values())
    assert np.all(bufs[2].download() == -5)  # nothing ran
    for z in bufs:
        z.free()


def test_calls_with_nothing_to_do(ctx):
    from aurora_amd.gpu import PagedBatch, PagedKvReadKernel, SampleKernel

    c = Case8(np.random.default_rng(14), [1], [5])
    dev = Device8(ctx, c)
    SampleKernel.new().dispatch_into(ctx, 0, 10, 0, 0, 0, 0, 10)
    SampleKernel.new().dispatch_into(ctx, 0, 100000, 0, 0, 0, 0, 100000)
    for batch, first, count in ((PagedBatch(0, 0, 0, 0, 0, 0, 1, 0), 0, 0), (dev.batch, 3, 0)):
        PagedKvReadKernel.new().dispatch_into(ctx, dev.cache, batch, dev.out.ptr, dev.out.ptr, 64, first, count)
    PagedKvReadKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, 64, 0, 5)
    assert np.all(dev.out.download() == 7.5)
    dev.free()


def test_one_page_of_two_sequences(ctx):
    """Sequences may read one page (a shared beginning); only one of them appends behind it, in a page of its own."""
    c = Case8(np.random.default_rng(15), [1, 2, 1], [20, 37, 33], 0, 16, 2, 2, 32, 8)
    c.pages[1, 0] = c.pages[2, 0] = c.pages[0, 0]
    dev = Device8(ctx, c)
    x = np.random.default_rng(1).standard_normal((c.n_tok, 64)).astype(np.float32)
    from aurora_amd.gpu import GpuBuffer

    new = GpuBuffer.from_slice(ctx, np.pad(x, ((0, 0), (0, 4))).ravel())
    q = GpuBuffer.from_slice(ctx, c.q.ravel())
    q_out = GpuBuffer.zeros(ctx, c.n_tok * (c.h * 32 + 4))
    _append(ctx, c, dev, q, new, new, 0, 0, 0, False, q_out)
    c.append(x.reshape(-1, 2, 32), x.reshape(-1, 2, 32))
    for a, w in zip(dev.bytes(), (c.kb, c.vb, c.ks, c.vs)):
        nan = (w & 127 == 127) & (w.ndim == 2)
        assert np.array_equal(a[~nan], w[~nan])
    dev.attend()
    out, _ = dev.result()
    want, _, tol, _ = attention_blocks(c)
    assert np.all(np.abs(out - want) <= tol)
    for z in (new, q, q_out):
        z.free()
    dev.free()


@pytest.mark.parametrize("dh", [8, 16, 32, 48, 64, 88, 128])
@pytest.mark.parametrize("block", [1, 2, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("kv", [1, 3])
def test_append_of_every_block(ctx, dh, block, kv):
    """Every number of waves that share a block: whole blocks, first and last parts of some, growing scales."""
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel

    rng = np.random.default_rng(dh + block)
    n, past = [150, 1, 40, 128], [0, 70, 100, 3]
    c = Case8(rng, n, [x + y for x, y in zip(n, past)], 0, 128, kv, 1, dh, block, behind=3)
    dev = Device8(ctx, c)
    row = kv * dh
    x = [(rng.standard_normal((c.n_tok, row)) * 2.0 ** rng.integers(-3, 4, (c.n_tok, 1))).astype(np.float32) for _ in range(2)]
    k, v = (GpuBuffer.from_slice(ctx, a.ravel()) for a in x)
    PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, k, v, row, 0, 0, 0, 0, 0, 0)
    with np.errstate(invalid="ignore"):
        c.append(*(a.reshape(-1, kv, dh) for a in x))
    got = dev.bytes()
    for a, w in zip(got[:2], (c.kb, c.vb)):
        nan = w & 127 == 127
        assert np.array_equal(a & 127 == 127, nan) and np.array_equal(a[~nan], w[~nan])
    assert np.array_equal(got[2], c.ks) and np.array_equal(got[3], c.vs)
    dev.free(), k.free(), v.free()


@pytest.mark.parametrize("b,kv,group,prefix,dh", [(200, 2, 4, 300, 64), (70, 1, 5, 700, 128), (150, 3, 1, 900, 24),
                                                  (20, 4, 16, 14500, 64), (20, 2, 16, 14500, 128)])
def test_prefixes_of_many_rows(ctx, b, kv, group, prefix, dh):
    """Prefixes read once for more than 128 rows, light ones by items of 64 rows beside the own ones, heavy ones by
    larger items."""
    rng = np.random.default_rng(b)
    c = Case8(rng, [1] * b, [1 + 7 * i % 40 for i in range(b)], prefix, 32, kv, group, dh, 8, behind=1)
    dev = Device8(ctx, c)
    dev.attend()
    out, lse = dev.result()
    want, want_lse, tol, tol_lse = attention_blocks(c)
    assert np.all(np.abs(out[:b] - want[:b]) <= tol[:b]) and np.all(np.abs(lse[:b] - want_lse[:b]) <= tol_lse[:b])
    dev.free()
