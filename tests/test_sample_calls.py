"""CPU checks of the scratch that the choice's Python object keeps."""
import ctypes as C

from aurora_amd.gpu import SampleKernel

PTR = 0x10000  # an address that nothing here reads


class Context:
    """Counts what a context is asked for; addresses of its own."""

    def __init__(self, base):
        self.next, self.allocated, self.freed, self.scratch = base, [], [], None

    def call(self, name, *args):
        if name == "aur_malloc":
            self.allocated.append((self.next, args[0]))
            C.cast(args[1], C.POINTER(C.c_void_p))[0] = self.next
            self.next += args[0]
        elif name == "aur_free":
            self.freed.append(args[0])
        else:
            assert name == "aur_sample"
            self.scratch = args[9:11]


def _call(kernel, ctx, b, vocab):
    ctx.scratch = None
    kernel.dispatch_into(ctx, PTR, vocab, PTR, PTR, 0, b, vocab)
    return ctx.scratch


def test_a_context_keeps_its_scratch():
    """One object in turn on two contexts, reserved on both: each call has its context's, and none allocates."""
    one, two, kernel = Context(1 << 20), Context(1 << 40), SampleKernel.new()
    n = kernel.scratch_bytes(64, 131072)
    kernel.reserve(one, 64, 131072), kernel.reserve(two, 64, 131072)
    for _ in range(10):
        for ctx in (one, two):
            assert _call(kernel, ctx, 64, 131072) == (ctx.allocated[0][0], n)
            assert _call(kernel, ctx, 3, 40000) == (ctx.allocated[0][0], n)  # less does not take another
    assert len(one.allocated) == len(two.allocated) == 1
    kernel.free()
    assert one.freed == [one.allocated[0][0]] and two.freed == [two.allocated[0][0]]


def test_a_growing_batch_keeps_little():
    """Row by row up to 64: a few allocations, whose sum stays below twice the last one's."""
    ctx, kernel = Context(1 << 20), SampleKernel.new()
    for b in range(1, 65):
        _, nbytes = _call(kernel, ctx, b, 131072)
        assert nbytes >= kernel.scratch_bytes(b, 131072)
    sizes = [n for _, n in ctx.allocated]
    assert len(sizes) <= 7 and sum(sizes) < 2 * sizes[-1] and sizes[-1] < 2 * kernel.scratch_bytes(64, 131072)
    kernel.free()
    assert sorted(ctx.freed) == sorted(p for p, _ in ctx.allocated)


def test_short_rows_take_none():
    ctx, kernel = Context(1 << 20), SampleKernel.new()
    assert _call(kernel, ctx, 64, 32768) == (0, 0) and not ctx.allocated
