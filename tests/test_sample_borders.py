"""The logits at which ranges and min_p's kept tokens end, found by the host's arithmetic: exactly, and after a bounded
number of looks, also where the border stands at 0, next to which floats are far denser than differences of logits."""
import math
import subprocess

import numpy as np
import pytest

from tests.paged_tiles import ROOT

# A guess and its neighbour; or up to 33 doublings and 32 halvings.
USUAL, MOST = 2, 66


@pytest.fixture(scope="module")
def borders(tmp_path_factory):
    exe = tmp_path_factory.mktemp("borders") / "borders"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(exe),
                    str(ROOT / "tests" / "cpp" / "sample_ranges.cpp")], check=True)

    def ask(lines):
        res = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, x)) for x in lines), capture_output=True, text=True,
                             check=True, timeout=60)
        rows = [x.split() for x in res.stdout.splitlines()]
        assert len(rows) == len(lines)
        return [(float.fromhex(a), int(b), int(c), int(n)) for a, b, c, n in rows]

    return ask


@pytest.mark.parametrize("m", [0.0, 0.140625, 1.984375, 3.0, -2.5, 15.984375, 6.0123, 1e-30, 1e30, -1e30, 3.4e38, -3.4e38])
@pytest.mark.parametrize("T", [1.0, 0.5, 0.75, 1.3, 1e-3, 1e-45, 100.0, 3e38])
def test_ranges(borders, m, T):
    got = borders([(repr(m), repr(T), 0.5, bin) for bin in range(1024)])
    edges = [a for a, *_ in got]
    assert all(b and c for _, b, c, _ in got) and max(n for *_, n in got) <= MOST
    assert all(x >= y for x, y in zip(edges, edges[1:])) and edges[-1] == -float(np.finfo(np.float32).max)


def test_a_border_at_zero(borders):
    """The border of range 63 below 1.984375 = 127/64 at T 1 stands at 0, where the result of m - v is the same for all
    |v| < 2^-54: the border is the first one above them."""
    (at, passes, ends, looked), = borders([(1.984375, 1.0, 0.5, 63)])
    assert passes and ends and 2.0**-54 <= at <= 2.0**-52 and looked <= MOST


@pytest.mark.parametrize("p", [1e-45, 1e-6, 0.01, 0.05, 0.367879450, 0.5, 0.999, 1.0])
def test_min_p(borders, p):
    rng = np.random.default_rng(1)
    p32 = float(np.float32(p))
    lines = []
    for T in (1.0, 0.7, 1e-3, 50.0, 1e30):
        zero = -T * math.log(p32)  # the largest logit that puts the border next to 0
        for m in [0.0, 1.0, -1.0, 20.0, float(np.float32(zero)), 1e30, *(rng.standard_normal(20) * 10).astype(np.float32)]:
            lines.append((repr(float(np.float32(m))), repr(T), repr(p32), -1))
    got = borders(lines)
    assert all(b and c for _, b, c, _ in got) and max(n for *_, n in got) <= MOST


def test_usual_borders_take_two_looks(borders):
    rng = np.random.default_rng(2)
    got = borders([(repr(float(np.float32(m))), repr(float(np.float32(T))), 0.5, int(b))
                   for m, T, b in zip(rng.uniform(4, 20, 500), rng.uniform(0.3, 2, 500), rng.integers(0, 1023, 500))])
    assert np.mean([n <= USUAL for *_, n in got]) > 0.9 and all(b and c for _, b, c, _ in got)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9000, 40000, 131072])
@pytest.mark.parametrize("by", ["top_k", "top_p", "min_p"])
def test_borders_at_zero_on_the_device(ctx, vocab, by):
    """Rows of bf16 logits whose largest is 127/64 and whose border lies in one of the ranges that end at 0."""
    from tests.test_sample_gpu import _check, _run

    rng = np.random.default_rng(vocab)
    b, m = 16, np.float32(127 / 64)
    x = np.clip(0.7 * rng.standard_normal((b, vocab)), -3, 1.97).astype(np.float32)
    x[:, 4000:] -= 9
    x = (x.view(np.uint32) & 0xffff0000).view(np.float32).copy()
    x[np.arange(b), rng.integers(0, vocab, b)] = m
    above = (x > 0).sum(1)
    w = np.exp((x - m).astype(np.float64))
    kw = {"top_k": dict(top_k=(above + np.arange(-20, 60, 5)).astype(np.int32)),
          "top_p": dict(top_p=((w * (x > 0)).sum(1) / w.sum(1) * (1 + np.linspace(-0.008, 0.008, b))).astype(np.float32)),
          "min_p": dict(min_p=np.exp(-m.astype(np.float64)) * (1 + 2.0**-24 * np.arange(-8, 8)))}[by]
    for v in kw.values():  # held to it: the last logit that a border keeps is next to 0
        for r in range(b):
            order = np.sort(x[r])[::-1]
            last = order[int(v[r]) - 1] if by == "top_k" else order[np.searchsorted(np.cumsum(np.sort(w[r])[::-1]), v[r] * w[r].sum())] \
                if by == "top_p" else 0.0
            assert abs(last) < 1 / 32, last
    u = rng.random(b).astype(np.float32)
    tokens, lp = _run(ctx, x, u, **kw)
    _check(x, u, tokens, lp, **kw)
