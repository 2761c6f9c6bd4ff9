"""Calls of the paged kernels that their documentation allows or refuses, next to those of
tests/test_paged_gpu.py."""
import numpy as np
import pytest

from tests.paged_ref import Case
from tests.paged_tiles import attention_blocks
from tests.test_paged_gpu import Device

pytestmark = pytest.mark.gpu


def test_one_buffer_of_two_strides_is_refused(ctx):
    """q rotated in place with rows of another stride would overwrite rows not yet read; a single row, and
    one stride, run."""
    from aurora_amd._lib import AuroraError
    from aurora_amd.gpu import PagedKvAppendKernel

    for n, refused in (([1, 1], True), ([2], True), ([1], False)):
        c = Case(np.random.default_rng(13), n, [17] * len(n), 30, 16, 2, 1, 64)
        dev = Device(ctx, c, ld_q=128 + 8)
        x = dev.q.ptr
        before = dev.q.download()

        def append(ld_qo):
            PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, x, 136, dev.out, dev.out, 128, x, ld_qo, 0,
                                                    0, 0, 2)

        if refused:
            with pytest.raises(AuroraError, match="one buffer"):
                append(128)
            assert np.array_equal(dev.q.download(), before, equal_nan=True)
        else:
            append(128)
        append(136)
        assert np.array_equal(dev.q.download(), before, equal_nan=True)  # no rotation: copied onto itself
        dev.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,prefix,group", [([1, 1, 1, 1], 100, 1), ([1] * 40, 2000, 1), ([9, 30, 2, 20], 100, 2),
                                            ([60, 70, 90, 80], 1500, 2)])
def test_values_beyond_the_bounds_touch_nothing_else(ctx, n, prefix, group, dtype):
    """Offsets and lengths that break the host's bounds, or are not ascending, are cut to them: other rows of the
    outputs and of the pools stay as they were, and sequences whose own values are sound keep their results."""
    from aurora_amd.gpu import GpuBuffer, PagedKvAppendKernel

    rng = np.random.default_rng(21)
    c = Case(rng, n, [x + 30 for x in n], prefix, 16, 2, group, 64, dtype, behind=5)
    dev = Device(ctx, c, ld_q=c.h * 64 + 4, ld_o=c.h * 64 + 4)
    want, want_lse, tol, tol_lse = attention_blocks(c)
    x = GpuBuffer.from_slice(ctx, rng.standard_normal(c.n_tok * 128).astype(np.float32))
    pools = [p.download() for p in (dev.k, dev.v)]
    named = np.zeros(c.n_pages * 16, bool)
    for s in range(c.b):
        for page in c.pages[s, :-(-c.length[s] // 16)]:
            named[page * 16:page * 16 + 16] = True
    off, length = c.off.copy(), c.length.astype(np.int32)
    for bad_off, bad_len in [({-1: c.n_tok + 1000}, {}), ({-1: 2**31 - 1}, {0: -5}), ({1: -2**31}, {1: 2**31 - 1}),
                             ({0: -7, -1: off[-2]}, {0: -2**31, 1: c.max_own + 1})]:
        o, l = off.copy(), length.copy()
        for i, v in bad_off.items():
            o[i] = v
        for i, v in bad_len.items():
            l[i] = v
        dev.off.upload(o)
        dev.len.upload(l)
        dev.out.upload(np.full(dev.out.len, 7.5, np.float32))
        dev.lse.upload(np.full(dev.lse.len, 7.5, np.float32))
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
        PagedKvAppendKernel.new().dispatch_into(ctx, dev.cache, dev.batch, 0, 0, x, x, 128, 0, 0, 0, 0, 0, 0)
        for have, was in zip((dev.k, dev.v), pools):
            have, was = (y.view(np.uint16).reshape(len(named), -1) for y in (have.download(), was))
            assert np.array_equal(have[~named], was[~named])
            changed = (have != was).any(1)
            for s in whole:  # a sound sequence's old rows stay, its new ones come
                rows = c.rows(c.pages[s], c.length[s])
                assert not changed[rows[:-n[s]]].any()
        for have, was in zip((dev.k, dev.v), pools):
            have.upload(was)
    x.free()
    dev.free()
