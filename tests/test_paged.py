"""CPU checks of the paged K/V cache: what the library refuses of a cache and a batch (the scratch
query runs the same checks as the launches, without a device), what the Python structs refuse, and the
float64 definitions the GPU tests compare with, against each other."""
import numpy as np
import pytest

from tests.paged_ref import Case, attention, from_bf16_bits, rotate, to_bf16_bits

PTR = 0x10000  # a 16-byte aligned address that nothing here reads


def _query(cache=None, batch=None, n_head=4):
    """(scratch bytes, the library's message) for a valid cache and batch with some fields replaced."""
    from aurora_amd import _lib
    from aurora_amd.gpu import PagedBatch, PagedKvCache

    c = dict(k=PTR, v=PTR, n_pages=64, page_len=16, n_kv_head=2, d_head=32, dtype="f32")
    b = dict(tok_off=PTR, own_len=PTR, pages=PTR, b=4, max_pages=64, n_tok=4, max_tok=1, max_own=1000,
             prefix_pages=PTR, n_prefix_pages=300, prefix_len=4096)
    c.update(cache or {})
    b.update(batch or {})
    cc, bb = PagedKvCache(**c), PagedBatch(**b)
    lib = _lib.load()
    n = lib.aur_mha_paged_ws_bytes(cc.ref, bb.ref, n_head)
    return n, lib.aur_last_error(None).decode() if n == 0 else ""


def test_scratch_of_a_valid_batch():
    n, _ = _query()
    assert n > 0 and n % (4 * 4 * 4 * (32 + 2)) == 0  # records of d_head + 2 floats for 4 tokens of 4 heads
    assert _query(batch=dict(prefix_len=0, max_own=16))[0] == 0  # one range of keys: no records


@pytest.mark.parametrize("cache,batch,what", [
    (dict(k=0), {}, "pools"),
    (dict(v=PTR + 8), {}, "16-byte"),
    (dict(n_pages=0), {}, "n_pages=0"),
    (dict(page_len=0), {}, "page_len=0"),
    (dict(page_len=24), {}, "power of two"),
    (dict(n_kv_head=0), {}, "n_kv_head=0"),
    (dict(d_head=0), {}, "d_head=0"),
    (dict(d_head=20), {}, "multiples of 8"),
    (dict(d_head=136), {}, "up to 128"),
    (dict(n_pages=1 << 28, page_len=16), {}, "pool of"),
    ({}, dict(tok_off=0), "null array"),
    ({}, dict(own_len=0), "null array"),
    ({}, dict(pages=0), "null array"),
    ({}, dict(prefix_pages=0), "null array"),
    ({}, dict(max_tok=0), "max_tok"),
    ({}, dict(max_own=64 * 16 + 1), "max_own=1025"),
    ({}, dict(prefix_len=300 * 16 + 1), "prefix_len=4801"),
    ({}, dict(prefix_len=1 << 30, n_prefix_pages=1 << 27), "prefix_len"),
    ({}, dict(n_tok=1 << 25), "n_tok"),
])
def test_refused_caches_and_batches(cache, batch, what):
    n, msg = _query(cache, batch)
    assert n == 0 and what in msg, msg


def test_python_structs_refuse():
    from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvCache, PagedMhaKernel

    with pytest.raises(ValueError, match="dtype"):
        PagedKvCache(PTR, PTR, 4, 16, 2, 32, "f16")
    short = GpuBuffer(None, PTR, 4 * 16 * 2 * 32 - 1, np.uint16)
    with pytest.raises(ValueError, match="pool"):
        PagedKvCache(PTR, short, 4, 16, 2, 32, "bf16")
    i32 = lambda n: GpuBuffer(None, PTR, n, np.int32)  # noqa: E731
    with pytest.raises(ValueError, match="tok_off"):
        PagedBatch(i32(4), i32(4), i32(8), 4, 2, 4, 1, 32)
    with pytest.raises(ValueError, match="pages"):
        PagedBatch(i32(5), i32(4), i32(7), 4, 2, 4, 1, 32)
    cache, batch = PagedKvCache(PTR, PTR, 4, 16, 2, 32), PagedBatch(i32(5), i32(4), i32(8), 4, 2, 4, 1, 32)
    with pytest.raises(ValueError, match="PagedMhaKernel out"):
        PagedMhaKernel().dispatch_into(None, cache, batch, PTR, 64, GpuBuffer(None, PTR, 4 * 64 - 1), 64, 0, PTR, 0, 2)


def test_definition_equals_causal_attention():
    """The paged definition on a prefix and tails equals plain causal attention over the whole sequence."""
    from tests.attn_ref import causal_attention_f64

    rng = np.random.default_rng(3)
    c = Case(rng, [5], [9], prefix=7, page=4, kv=3, dh=8)
    out, lse, _, _ = attention(c)
    k, v, there = c.keys(0)
    assert there.all() and len(k) == 16
    q = rng.standard_normal((16, 3, 8))
    q[11:] = c.q.reshape(5, 3, 8)
    want, want_lse = causal_attention_f64(q[None], k[None], v[None])
    np.testing.assert_allclose(out.reshape(5, 3, 8), want[0, 11:], rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(lse, want_lse[0].T[11:], rtol=1e-12)


def test_rotation_keeps_relative_positions():
    """q·k after rotation depends on the positions' difference alone, and lengths stay."""
    rng = np.random.default_rng(4)
    q, k = rng.standard_normal((1, 32)), rng.standard_normal((1, 32))
    for pairs in (False, True):
        a = [float((rotate(q, [p + 9], 1, 32, 24, pairs) * rotate(k, [p], 1, 32, 24, pairs)).sum()) for p in (0, 5, 1000)]
        np.testing.assert_allclose(a, a[0], rtol=1e-11)
        np.testing.assert_allclose(np.linalg.norm(rotate(q, [77], 1, 32, 24, pairs)), np.linalg.norm(q), rtol=1e-13)


def test_bf16_rounding_is_to_nearest_even():
    x = np.array([1.0, 1.00390625, 1.01171875, -2.5, 3e38, 1e-40], np.float32)  # 1 + 2^-8: a tie, to 1
    got = from_bf16_bits(to_bf16_bits(x))
    assert got[0] == 1.0 and got[1] == 1.0 and got[2] == 1.015625
    assert np.all(np.abs(got[:5] - x[:5]) <= 2.0**-8 * np.abs(x[:5]))
