"""Calls of the paged kernels that their documentation allows or refuses, next to those of
tests/test_paged_gpu.py."""
import numpy as np
import pytest

from tests.paged_ref import Case
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
