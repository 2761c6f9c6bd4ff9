"""CPU checks of how the paged attention cuts calls into items (aurora_amd/csrc/paged_plan.hpp, compiled
here by itself): the batches that the GPU tests of its kernels run reach the kernels that they are
meant for, and all of them.  A planner that sends one elsewhere fails here, and wants batches for what
it left out."""
import subprocess

import numpy as np
import pytest

from tests.paged_ref import Case, attention
from tests.paged_tiles import ALL, D_HEADS, OWN, POOLED, ROOT, attention_blocks, every_kernel, kernels

FIELDS = "pooled p_tile p_tiles p_splits o_tile o_tiles o_splits step_rows head_tiles".split()


@pytest.fixture(scope="module")
def plan_of(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "paged_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(exe),
                    str(ROOT / "tests" / "cpp" / "paged_plan.cpp")], check=True, capture_output=True, text=True)

    def plans(calls):
        """calls: (b, n_tok, max_tok, max_own, prefix_len, n_kv_head, group, d_head, f32)."""
        text = "\n".join(" ".join(str(int(x)) for x in c) for c in calls)
        res = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True, timeout=60)
        return [dict(zip(FIELDS, map(int, line.split()))) for line in res.stdout.splitlines()]

    return plans


def _call(b, dh, f32):
    return len(b.n), sum(b.n), max(b.n), max(b.length), b.prefix, b.kv, b.group, dh, f32


@pytest.mark.parametrize("name", ALL)
def test_batches_reach_their_items(plan_of, name):
    b = ALL[name]
    for f32 in (True, False):
        for dh, p in zip(D_HEADS, plan_of([_call(b, dh, f32) for dh in D_HEADS])):
            want = b.narrow if dh <= 64 else b.wide
            assert (p["p_tile"], p["o_tile"]) == want, (dh, f32, p)
            assert p["pooled"] == (name in POOLED)
            assert (p["p_splits"] + p["o_splits"] > 1) == b.cut, (dh, f32, p)
            if name.startswith("several"):
                assert p["o_tiles"] > 1


def test_every_kernel_is_reached(plan_of):
    for f32 in (True, False):
        got = set()
        for b in ALL.values():
            for p in plan_of([_call(b, dh, f32) for dh in D_HEADS]):
                got |= kernels(p)
        assert got == every_kernel(f32), (every_kernel(f32) - got, got - every_kernel(f32))


def test_plans_hold_every_key_and_row(plan_of):
    """Over random sizes: tiles hold all rows, ranges are at most as many as a join reads, and the
    items fit a launch wherever the scratch query accepts the call."""
    rng = np.random.default_rng(1)
    calls = []
    for _ in range(3000):
        b = int(2 ** rng.uniform(0, 12))
        max_tok = 1 if rng.random() < 0.4 else int(2 ** rng.uniform(0, 13))
        n_tok = int(rng.integers(max_tok, b * max_tok + 1))
        calls.append((b, n_tok, max_tok, int(rng.choice([0, 2 ** rng.uniform(0, 20)])),
                      int(rng.choice([0, 2 ** rng.uniform(0, 20)])), rng.integers(1, 17), rng.choice([1, 2, 3, 4, 8, 16]),
                      8 * rng.integers(1, 17), rng.random() < 0.5))
    for c, p in zip(calls, plan_of(calls)):
        b, n_tok, max_tok, max_own, prefix, kv, g, dh, f32 = (int(x) for x in c)
        assert p["o_tile"] * p["o_tiles"] >= max_tok * g and p["o_tile"] in (16, 64, 128, 256), (c, p)
        assert 1 <= p["o_splits"] <= 48 and p["p_splits"] <= 48, (c, p)
        assert p["o_tile"] != 256 or dh <= 64
        if p["pooled"]:
            assert prefix > 0 and p["p_splits"] >= 1 and p["p_tile"] * p["p_tiles"] >= n_tok * g, (c, p)
            assert p["p_tile"] == 64 or p["o_tile"] <= 16 or p["p_tile"] > 64  # one launch: tiles of one kind
            assert p["o_tile"] <= 64
        else:
            assert p["p_tiles"] == p["p_splits"] == 0
        assert p["step_rows"] in ((1, 2, 4, 16) if f32 else (1, 2, 16))
        assert p["step_rows"] >= (g if max_tok == 1 and g <= 16 else 1)


@pytest.mark.parametrize("seed", range(6))
def test_the_blocked_definition_equals_the_plain_one(seed):
    rng = np.random.default_rng(seed)
    b = int(rng.integers(1, 5))
    n = rng.integers(0, 9, b)
    n[0] = max(n[0], 1)
    length = np.maximum(n + rng.integers(-3, 30, b), 0)
    c = Case(rng, n, length, int(rng.choice([0, 1, 33])), 8, 2, int(rng.choice([1, 3])), 16, behind=1)
    if seed % 2 and c.prefix:
        c.prefix_pages[0] = -1
    if length[0]:
        c.pages[0, 0] = c.n_pages
    for x, y in zip(attention(c), attention_blocks(c)):
        np.testing.assert_allclose(y, x, rtol=1e-11, atol=1e-300)


def test_infinities_in_the_blocked_definition():
    rng = np.random.default_rng(9)
    c = Case(rng, [5, 1, 3], [9, 30, 4], 11, 8, 2, 2, 16, behind=1)
    own = [c.rows(c.pages[s], c.length[s]) for s in range(3)]
    c.vp[own[0][6], 3], c.vp[own[1][20], 20] = np.inf, np.nan
    c.vp[own[0][8], 3] = -np.inf
    c.kp[own[2][2], 5], c.kp[own[0][8], 20] = np.inf, np.nan
    c.kp[c.prefix_pages[0] * 8 + 3, 9] = -np.inf
    with np.errstate(all="ignore"):
        want, lse, tol, _ = attention(c)
        got, got_lse, got_tol, _ = attention_blocks(c)
    np.testing.assert_allclose(got, want, rtol=1e-11, atol=1e-300)
    np.testing.assert_allclose(got_lse, lse, rtol=1e-11)
    bounded = np.isfinite(tol) & np.isfinite(want)
    np.testing.assert_allclose(got_tol[bounded], tol[bounded], rtol=1e-11)
    assert np.isnan(want).any() and np.isinf(want).any() and bounded.any()


def test_a_mistake_in_the_definition_shows():
    """A mask one key too far, or a key that is not the cached one, lies outside the bounds that the kernels
    are held to (but in rows where that key has next to no weight); the order of keys does not."""
    b = OWN["128 rows"]
    c = b.case(24, "f32")
    want, _, tol, _ = attention_blocks(c)
    c.length[0] += 1
    c.kp[np.isnan(c.kp)] = c.vp[np.isnan(c.vp)] = 0.5
    far = (np.abs(attention_blocks(c)[0] - want) > 2 * tol).any(1)
    assert far[:c.off[1]].mean() > 0.9 and not far[c.off[1]:].any()
    c = b.case(24, "f32")
    c.prefix_pages[[3, 50]] = c.prefix_pages[[50, 3]]
    assert np.all(np.abs(attention_blocks(c)[0] - want) <= 1e-3 * tol)
    c.kp[c.prefix_pages[7] * c.page] *= 1.5
    assert (np.abs(attention_blocks(c)[0] - want) > 2 * tol).any(1).mean() > 0.9
