"""CPU checks of what the paged kernels' Python calls hand to the library."""
import ctypes as C

import numpy as np
import pytest

from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvAppendKernel, PagedKvCache, PagedMhaKernel

PTR = 0x10000  # an address that nothing here reads


class Named(GpuBuffer):
    """A program's own kind of buffer."""


class Recorder:
    def __init__(self):
        self.args = None

    def call(self, name, *args):
        self.args = args


def _set_up():
    i32 = lambda n: Named(None, PTR, n, np.int32)  # noqa: E731
    cache = PagedKvCache(Named(None, PTR, 4096), Named(None, PTR, 4096), 4, 16, 2, 32)
    return cache, PagedBatch(i32(5), i32(4), i32(8), 4, 2, 4, 1, 32)


@pytest.mark.parametrize("buffer", [GpuBuffer, Named])
@pytest.mark.parametrize("which", range(4))
def test_any_kind_of_buffer_is_unwrapped(buffer, which):
    """One buffer among raw pointers, of the class itself or of one derived from it."""
    cache, batch = _set_up()
    long = buffer(None, PTR + 64, 4096)
    ctx, x = Recorder(), [PTR] * 4
    x[which] = long
    PagedKvAppendKernel().dispatch_into(ctx, cache, batch, x[0], 128, x[1], x[2], 64, PTR, 128, x[3], 32, 32, 4)
    assert ctx.args[2] == (PTR + 64 if which == 0 else PTR) and all(isinstance(a, (int, float)) for a in ctx.args)
    PagedMhaKernel().dispatch_into(ctx, cache, batch, x[0], 128, x[1], 128, x[2], x[3], 4096, 4)
    assert (PTR + 64) in ctx.args and all(isinstance(a, int) for a in ctx.args)


@pytest.mark.parametrize("buffer", [GpuBuffer, Named])
@pytest.mark.parametrize("which,what", [(0, "PagedMhaKernel q"), (1, "PagedMhaKernel out"), (2, "PagedMhaKernel lse"),
                                        (3, "PagedMhaKernel scratch")])
def test_any_kind_of_buffer_is_checked(buffer, which, what):
    cache, batch = _set_up()
    x = [PTR] * 4
    x[which] = buffer(None, PTR, 15)
    with pytest.raises(ValueError, match=what):
        PagedMhaKernel().dispatch_into(Recorder(), cache, batch, x[0], 128, x[1], 128, x[2], x[3], 4096, 4)


@pytest.mark.parametrize("buffer", [GpuBuffer, Named])
@pytest.mark.parametrize("which,what", [(0, "PagedKvAppendKernel q"), (1, "PagedKvAppendKernel k/v"),
                                        (2, "PagedKvAppendKernel k/v"), (3, "PagedKvAppendKernel q_out"),
                                        (4, "PagedKvAppendKernel table")])
def test_any_kind_of_buffer_is_checked_by_the_append(buffer, which, what):
    cache, batch = _set_up()
    x = [PTR] * 5
    x[which] = buffer(None, PTR, 15)
    with pytest.raises(ValueError, match=what):
        PagedKvAppendKernel().dispatch_into(Recorder(), cache, batch, x[0], 128, x[1], x[2], 64, x[3], 128, x[4], 32, 32,
                                            4)


def test_raw_pointers_pass_as_they_are():
    """Addresses, ctypes pointers and None (no q, no lse) reach the library as they came."""
    cache, batch = _set_up()
    ctx, void = Recorder(), C.c_void_p(PTR)
    PagedKvAppendKernel().dispatch_into(ctx, cache, batch, None, 0, void, PTR, 64, None, 0, None, 0, 0, 0)
    assert ctx.args[2:4] == (None, 0) and ctx.args[4] is void and ctx.args[7] is None
    PagedMhaKernel().dispatch_into(ctx, cache, batch, void, 128, PTR, 128, None, None, 0, 4)
    assert ctx.args[2] is void and ctx.args[6] is None


def test_a_refused_type_allocates_nothing():
    ctx = Recorder()
    with pytest.raises(ValueError, match="f16"):
        PagedKvCache.zeros(ctx, 4, 16, 2, 32, "f16")
    assert ctx.args is None
