"""The paged attention's kernels, each by batches that the plan gives to it (tests/paged_tiles.py; which
batch reaches what is held on the CPU by tests/test_paged_plan.py), against the definition in float64."""
import ctypes

import numpy as np
import pytest

from tests.paged_tiles import ALL, D_HEADS, attention_blocks
from tests.test_paged_gpu import Device, _hip

pytestmark = pytest.mark.gpu


def _compare(c, out, lse, loss=0.0, what=""):
    """Every row against the definition: the same infinities and NaN, the rest within the bounds."""
    want, want_lse, tol, tol_lse = attention_blocks(c, loss)
    d, n = c.h * c.dh, int(c.off[-1])
    assert np.all(out[n:] == 7.5) and np.all(out[:, d:] == 7.5), f"{what}: rows or columns that are none were written"
    assert np.all(lse[n:] == 7.5)
    worst = 0.0
    for have, want, tol in ((out[:n, :d], want[:n], tol[:n]), (lse[:n], want_lse[:n], tol_lse[:n])):
        fine = np.isfinite(want)
        assert fine.any()
        assert np.array_equal(np.isnan(have), np.isnan(want)), what
        assert np.array_equal(have[np.isinf(want)], want[np.isinf(want)]), what
        err = np.abs(have[fine] - want[fine])
        worst = max(worst, float((err / np.maximum(tol[fine], 1e-300)).max()))
        assert worst <= 1.0, f"{what}: {worst} of the bound"
    return worst


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dh", D_HEADS)
@pytest.mark.parametrize("name", ALL)
def test_every_kernel_matches_float64(ctx, name, dh, dtype):
    """Rows of other strides than their length and a row behind the last sequence; and the same bits from a
    second call, whose scratch holds the first one's records."""
    b = ALL[name]
    c = b.case(dh, dtype, behind=1)
    dev = Device(ctx, c, ld_q=c.h * dh + 8, ld_o=c.h * dh + 4)
    dev.attend()
    out, lse = dev.result()
    print(f"[paged] {_compare(c, out, lse):.3f} of the bound")
    dev.attend()
    for x, y in zip((out, lse), dev.result()):
        assert np.array_equal(x, y)
    dev.free()


HARD = ["64 rows", "64 rows, group 4", "128 rows", "128 rows, group 2", "256 rows", "several tiles", "prefix 64, own 64",
        "one prompt among steps", "prefix 64, own 16", "prefix 256, own 16", "prefix 256, own 64", "prefix 16, own 16"]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dh", [40, 64, 128])
@pytest.mark.parametrize("name", HARD)
@pytest.mark.parametrize("where", ["own", "prefix"])
def test_infinities_of_many_rows(ctx, where, name, dh, dtype):
    """Infinities and NaN among the keys and values of a batch: rows that see them get what the formula
    gives, rows of the same item that do not are as if they were not there."""
    c = ALL[name].case(dh, dtype)
    if where == "own":
        first, last = c.rows(c.pages[0], c.length[0]), c.rows(c.pages[-1], c.length[-1])
        mid = first[c.length[0] - c.n[0] + c.n[0] // 2]  # a new token's, that the ones before it do not see
        c.vp[mid, 3], c.vp[mid, dh + 6] = np.inf, np.nan
        c.vp[first[-1], 5], c.kp[first[-1], dh + 1] = -np.inf, np.nan
        c.kp[last[-1], 2] = np.inf  # the sign of the query's column decides: NaN, or a key without weight
    else:
        page = c.prefix_pages[c.prefix // c.page // 2] * c.page
        c.vp[page, 1], c.vp[page, 2] = np.inf, -np.inf
        c.vp[c.prefix_pages[0] * c.page, dh + 4] = np.nan
        c.kp[page, dh + 7] = -np.inf
    dev = Device(ctx, c)
    dev.attend()
    _compare(c, *dev.result())
    dev.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", HARD)
@pytest.mark.parametrize("vs,ks", [(2.0**-100, 1.0), (2.0**100, 1.0), (1.0, 2.0**40), (1.0, 2.0**-40)])
def test_values_of_any_size_in_tiles(ctx, vs, ks, name, dtype):
    """V of any size, and columns of K far larger or smaller than the others whose queries make up for it:
    nothing is lost beside a larger neighbour."""
    c = ALL[name].case(64, dtype)
    c.vp[:, ::2] *= np.float32(vs)
    _scale_columns(c, ks)
    dev = Device(ctx, c)
    dev.attend()
    _compare(c, *dev.result())
    dev.free()


def _scale_columns(c, ks):
    """Every third column of each head of K times ks, of the queries by 1/ks."""
    c.kp.reshape(len(c.kp), c.kv, c.dh)[:, :, 1::3] *= np.float32(ks)
    c.q.reshape(c.n_tok, c.h, c.dh)[:, :, 1::3] /= np.float32(ks)


LEAST = 2.0**-126  # the smallest normal number: the matrix cores take smaller bf16 operands as zero
FEW = ["one row", "two rows", "three rows", "16 rows of one sequence", "prefix 16, own 16"]  # no item of more than 16 rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", HARD + [x for x in FEW if x not in HARD] + ["prefix 64, own 1"])
@pytest.mark.parametrize("vs,ks", [(1.0, 2.0**-115), (1.0, 2.0**115), (2.0**-115, 1.0), (2.0**-130, 1.0), (2.0**-130, 2.0**-120)])
def test_values_next_to_the_smallest(ctx, vs, ks, name, dtype):
    """Keys, queries and values whose bf16 parts fall below 2^-126 are exact to 2^-126 (as is bf16's own
    rounding of the pools here); fp32 ones in items of up to 16 rows to their roundings, as any others."""
    c = ALL[name].case(64, dtype, seed=1)
    c.vp[:, ::2] *= np.float32(vs)
    _scale_columns(c, ks)
    dev = Device(ctx, c)
    dev.attend()
    _compare(c, *dev.result(), loss=0.0 if dtype == "f32" and name in FEW else LEAST)
    dev.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dh", [48, 128])
@pytest.mark.parametrize("name", HARD)
@pytest.mark.parametrize("own", ["some", "none"])
def test_pages_that_are_not_there_in_tiles(ctx, own, name, dh, dtype):
    """Page numbers outside the pool, the largest and smallest among them, take their keys out: single pages of
    the prefix and of the sequences; a sequence that keeps its last pages only, or none of its own."""
    c = ALL[name].case(dh, dtype)
    odd = [-1, c.n_pages, 2**31 - 1, -2**31, c.n_pages + 7]
    c.prefix_pages[[3, 7, 20, len(c.prefix_pages) // 2, -1]] = odd
    used = -(-c.length // c.page)
    for i, s in enumerate(np.flatnonzero(used > 0)):
        if i == 1:
            continue  # this one is whole
        c.pages[s, used[s] // 2] = odd[i % 5]
    longest = int(np.argmax(used))
    if own == "some":
        c.pages[longest, :(used[longest] + 1) // 2] = 2**31 - 1
    else:
        c.pages[longest] = -7
    dev = Device(ctx, c)
    dev.attend()
    _compare(c, *dev.result())
    dev.free()


def test_tiles_captured_into_a_graph(ctx):
    """Two batches, one with its prefix in a launch of its own, captured into one graph on one scratch;
    every replay, with eager calls in between and other queries and lengths, equals the eager calls."""
    from aurora_amd.gpu import GpuBuffer
    from aurora_amd._lib import load

    hip, stream = _hip(), load().aur_stream(ctx.ptr)
    cases = [ALL["prefix 256, own 64"].case(64, "f32"), ALL["128 rows"].case(64, "bf16")]
    eager, replayed = [[Device(ctx, c) for c in cases] for _ in range(2)]
    ws = GpuBuffer.zeros(ctx, max(d.ws_len for d in replayed))
    rng = np.random.default_rng(3)
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(stream, 1) == 0  # hipStreamCaptureModeThreadLocal
    try:
        for d in replayed:
            d.attend(ws=ws)
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    try:
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for step in range(4):
            q = [rng.standard_normal(d.q.len).astype(np.float32) for d in eager]
            for side in (eager, replayed):
                for d, x in zip(side, q):
                    d.q.upload(x)
                    d.len.upload((d.c.length - min(step, 1) * (d.c.length > 3)).astype(np.int32))
            for d in eager:
                d.attend()
            ctx.sync()
            assert hip.hipGraphLaunch(exe, stream) == 0
            ctx.sync()
            for x, y in zip(eager, replayed):
                for a, b in zip(x.result(), y.result()):
                    assert np.array_equal(a, b), step
    finally:
        if exe.value:
            hip.hipGraphExecDestroy(exe)
        if graph.value:
            hip.hipGraphDestroy(graph)
        for d in eager + replayed:
            d.free()
        ws.free()
