"""CPU checks of the 8-bit paged cache and of choosing tokens: what is refused, and the definitions that the
GPU tests compare with, against each other."""
import numpy as np
import pytest

from aurora_amd.gpu import GpuBuffer, PagedBatch, PagedKvCache, PagedKvReadKernel, SampleKernel
from tests.e4m3_ref import LEAST, MOST, NUMBERS, Case8, least_exponent, nearest, sample, sample_exact

PTR = 0x10000  # a 16-byte aligned address that nothing here reads


def _query(**fields):
    """The library's message for an e4m3 cache with some fields replaced ("" where it is taken)."""
    from aurora_amd import _lib

    c = PagedKvCache(PTR, PTR, 64, 16, 2, 32, "e4m3", PTR, PTR, 16)
    b = PagedBatch(PTR, PTR, PTR, 4, 64, 4, 1, 1000, PTR, 300, 4096)
    for name, x in fields.items():
        setattr(c._struct, name, x)
    lib = _lib.load()
    n = lib.aur_mha_paged_ws_bytes(c.ref, b.ref, 4)
    return "" if n else lib.aur_last_error(None).decode()


def test_an_e4m3_cache_is_taken():
    assert _query() == "" and _query(scale_len=1) == "" and _query(page_len=128, scale_len=128) == ""


@pytest.mark.parametrize("fields,what", [
    (dict(k_scale=0), "both scales"), (dict(v_scale=0), "both scales"), (dict(scale_len=0), "scale_len=0"),
    (dict(scale_len=12), "power of two"), (dict(scale_len=32), "up to page_len=16"),
    (dict(page_len=256, scale_len=256), "up to 128"), (dict(dtype=3), "dtype 3"), (dict(d_head=20), "multiples of 8"),
])
def test_refused_caches(fields, what):
    assert what in _query(**fields)


def test_other_types_do_not_look_at_the_scales():
    assert _query(dtype=0, k_scale=0, v_scale=0, scale_len=77) == "" and _query(dtype=1, scale_len=0) == ""


def test_python_structs_refuse():
    u8 = lambda n: GpuBuffer(None, PTR, n, np.uint8)  # noqa: E731
    n, s = 4 * 16 * 2 * 32, 4 * 2 * 4
    PagedKvCache(u8(n), u8(n), 4, 16, 2, 32, "e4m3", u8(s), u8(s), 4)
    for args, what in (((u8(n - 1), u8(n), 4, 16, 2, 32, "e4m3", u8(s), u8(s), 4), "pool"),
                       ((u8(n), u8(n), 4, 16, 2, 32, "e4m3", u8(s), u8(s - 1), 4), "scales"),
                       ((u8(n), u8(n), 4, 16, 2, 32, "e4m3", u8(s), None, 4), "k_scale and v_scale"),
                       ((u8(n), u8(n), 4, 16, 2, 32, "e4m3", u8(s), u8(s), 5), "scale_len 5"),
                       ((u8(n), u8(n), 4, 16, 2, 32, "e4m3", u8(s), u8(s), 32), "scale_len 32"),
                       ((u8(n), u8(n), 4, 16, 2, 32, "e4m3", u8(s), u8(s)), "scale_len 0"),
                       ((PTR, PTR, 4, 16, 2, 32, "bf16", PTR, PTR, 4), "k_scale and v_scale")):
        with pytest.raises(ValueError, match=what):
            PagedKvCache(*args)

    class Nothing:
        def call(self, *args):
            raise AssertionError(args)

    with pytest.raises(ValueError, match="scale_len"):
        PagedKvCache.zeros(Nothing(), 4, 16, 2, 32, "e4m3")
    f32 = lambda n: GpuBuffer(None, PTR, n)  # noqa: E731
    i32 = lambda n: GpuBuffer(None, PTR, n, np.int32)  # noqa: E731
    cache, batch = PagedKvCache(PTR, PTR, 4, 16, 2, 32), PagedBatch(PTR, i32(4), i32(8), 4, 2, 0, 0, 32)
    with pytest.raises(ValueError, match="k_out/v_out"):
        PagedKvReadKernel().dispatch_into(Nothing(), cache, batch, f32(4 * 10 * 64 - 1), 0, 64, 0, 10)
    ok = dict(logits=f32(2 * 10), u=f32(2), tokens=i32(2), logprob=f32(2), temperature=f32(2), top_k=i32(2), top_p=f32(2), min_p=f32(2))
    for name in ok:
        x = dict(ok, **{name: GpuBuffer(None, PTR, ok[name].len - 1, ok[name].dtype)})
        with pytest.raises(ValueError, match="SampleKernel"):
            SampleKernel().dispatch_into(Nothing(), x["logits"], 10, x["u"], x["tokens"], x["logprob"], 2, 10, x["temperature"],
                                         x["top_k"], x["top_p"], x["min_p"])
    with pytest.raises(AssertionError, match="aur_sample"):
        SampleKernel().dispatch_into(Nothing(), ok["logits"], 10, ok["u"], ok["tokens"], 0, 2, 10)


def test_scratch_of_the_choice():
    assert SampleKernel.scratch_bytes(64, 32768) == 0 and SampleKernel.scratch_bytes(0, 100000) == 0
    n = SampleKernel.scratch_bytes(3, 32769)
    assert n >= 3 * 3 * 1024 * 12 and n % 16 == 0
    assert SampleKernel.scratch_bytes(64, 131072) < 8 << 20  # less than a fourth of the logits


def test_numbers_and_rounding():
    import torch

    assert NUMBERS[126] == 448 and NUMBERS[1] == 2.0**-9 and np.isnan(NUMBERS[127]) and NUMBERS[8] == 2.0**-6
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.standard_normal(20000) * 100, rng.standard_normal(20000) * 0.01, np.arange(-448, 448, 0.25),
                        np.arange(-64, 64) * 2.0**-10, [0.0, -0.0, 448.0, 464.0, 1e30, np.nan, np.inf]])
    want = torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    got = nearest(x.astype(np.float32).astype(np.float64))
    fine = np.isfinite(x)
    assert np.array_equal(got[fine], want[fine]) and np.all(got[~fine] & 127 == 127)


def test_least_exponent():
    assert least_exponent(np.array([448.0])) == 0 and least_exponent(np.array([448.0001])) == 1
    assert least_exponent(np.zeros(3)) == LEAST and least_exponent(np.array([3.4e38, np.inf])) == MOST
    assert least_exponent(np.array([np.nan, 1.75])) == -8 and least_exponent(np.array([1.7500001])) == -7


def test_append_definition_keeps_values():
    """Every appended value stands within half a step of its number, in a block of any age."""
    rng = np.random.default_rng(2)
    c = Case8(rng, [9, 30], [20, 30], 0, 16, 2, 1, 32, 8)
    k, v = (rng.standard_normal((39, 2, 32)).astype(np.float32) for _ in range(2))
    c.append(k, v)
    for s in range(2):
        rows = c.rows(c.pages[s], c.length[s])[c.length[s] - c.n[s]:]
        for x, held in ((k, c.kp), (v, c.vp)):
            new = x[c.off[s]:c.off[s + 1]].reshape(-1, 64)
            assert np.all(np.abs(held[rows] - new) <= 2.0**-4 * np.abs(new) + 2.0**-10 * 2.0**-6)


def test_sample_definitions_agree():
    rng = np.random.default_rng(3)
    for _ in range(200):
        n = int(rng.integers(1, 40))
        w = rng.integers(1, 20, n)
        k, p, u = int(rng.integers(0, n + 1)), float(rng.choice([0.3, 0.77, 1.0])), float(rng.random())
        x = np.log(w)
        order = sorted(range(n), key=lambda i: (-w[i], i))
        a, lp, near = sample(x, u, 1.0, k if k < n else 0, p)
        if near > 1e-9:
            assert a == (order[0] if k == 1 else sample_exact([int(i) for i in w], order, k, p, u))
    # all of it: the token's share
    a, lp, _ = sample(np.log([1.0, 2.0, 5.0]), 0.3)
    assert a == 1 and abs(lp - np.log(2 / 8)) < 1e-12


def test_every_kernel_is_reached(tmp_path):
    """The batches that the GPU tests run on 8-bit pools reach all kernels, as the planner cuts them."""
    import subprocess

    from tests.paged_tiles import ALL, D_HEADS, ROOT, every_kernel, kernels
    from tests.test_paged_plan import FIELDS

    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(exe),
                    str(ROOT / "tests" / "cpp" / "paged_plan_e4m3.cpp")], check=True)
    calls = [(len(b.n), sum(b.n), max(b.n), max(b.length), b.prefix, b.kv, b.group, dh) for b in ALL.values() for dh in D_HEADS]
    res = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in calls), capture_output=True, text=True,
                         check=True, timeout=60)
    got = set()
    for line in res.stdout.splitlines():
        got |= kernels(dict(zip(FIELDS, map(int, line.split()))))
    assert got == every_kernel(False), (every_kernel(False) - got, got - every_kernel(False))
