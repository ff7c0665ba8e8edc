"""GPU: pkcu_sample_rows against its definition in 64 bits.

Tokens have to be equal: the kernel's weights are within 2^-44 of the largest and
2e-13 of their own value, so a running sum is off by less than 1e-12 of the total
and a uniform u falls that close to one of V borders in fewer than one row in
10^6. Log-probabilities: the exponent rounds in fp64, log1p of the other
weights' sum in fp32 (off by at most 3 steps of 2^-24 of its value), the
difference once: 2^-24 |logp| + 4 x 2^-24 log(S)."""
import math

import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu, f64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def plain(x, u, T, k, p, mp):
    """(token, log-probability, log of the kept weight over the largest) of one
    row of float64 values."""
    x = np.where(np.isnan(x), -np.inf, x)
    valid = x > -np.inf
    if not valid.any():
        return -1, -np.inf, 0.0
    top = x.max()
    if not T > 0:
        return int(np.argmax(x)), 0.0, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(x == top, 0.0, x - top)
        y = np.where(d == 0, 0.0, np.where(valid, d / T, -np.inf))
        if np.isinf(top):
            y = np.where(x == top, 0.0, -np.inf)
    w = np.exp(y)
    by = np.argsort(-x, kind="stable")[: int(valid.sum())]
    if k > 0:
        by = by[:k]
    if p < 1:
        c = np.cumsum(w[by])
        by = by[: 1 + int(np.searchsorted(c, max(p, 0.0) * c[-1], side="left"))]
    if mp > 0:
        by = by[w[by] >= min(mp, 1.0)]
    by = np.sort(by)
    c = np.cumsum(w[by])
    u = u if u > 0 else 0.0
    at = int(np.searchsorted(c, u * c[-1], side="right"))
    if at >= len(by):   # u from 1 on: the last that weighs something
        at = int(np.flatnonzero(w[by] > 2.0 ** -45)[-1])
    return int(by[at]), float(y[by[at]] - math.log(c[-1])), math.log(c[-1])


def check(cuda, logits, u, T=None, k=None, p=None, mp=None, what="", **kw):
    import torch
    rows, V = logits.shape
    tok = empty(rows, torch.int32).fill_(-7)
    lp = empty(rows).fill_(9.0)
    dev = lambda a, t="f32": None if a is None else (cu(a.astype(np.float32)) if t == "f32" else cu(a.astype(np.int32)))
    cuda.sample_rows(logits, dev(u), tok, lp, temperature=dev(T), top_k=dev(k, "i32"), top_p=dev(p), min_p=dev(mp), **kw)
    x, got, glp = f64(logits), f64(tok), f64(lp)
    at = lambda a, i, d: d if a is None else float(np.float32(a[i]))
    for i in range(rows):
        t, l, s = plain(x[i], at(u, i, 0), at(T, i, 1.0), 0 if k is None else int(k[i]), at(p, i, 1.0), at(mp, i, 0.0))
        assert got[i] == t, f"{what} row {i}: token {got[i]} instead of {t}"
        if t < 0:
            assert glp[i] == -np.inf
        else:
            assert abs(glp[i] - l) <= U * abs(l) + 4 * U * s + 1e-12, f"{what} row {i}: {glp[i]} instead of {l}"
    return tok, lp


def settings(rng, rows, mode):
    T = rng.uniform(0.5, 1.5, rows)
    k = rng.integers(1, 100, rows)
    p = rng.uniform(0.3, 0.99, rows)
    mp = rng.uniform(0.01, 0.3, rows)
    if mode == "mixed":
        k[::3] = 0
        p[1::3] = 1.0
        mp[::2] = 0.0
        T[5::7] = 0.0
    return dict(T=T, k=k if mode in ("top_k", "mixed") else None, p=p if mode in ("top_p", "mixed") else None,
                mp=mp if mode in ("min_p", "mixed") else None)


SHAPES = [(1, 1), (3, 2), (40, 33), (70, 100), (300, 1025), (9, 4097), (150, 5000), (20, 32000), (1, 131072), (2, 131072),
          (30, 65536), (1, 262144), (3, 262144)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mode", ["plain", "top_k", "top_p", "min_p", "mixed"])
@pytest.mark.parametrize("rows,V", SHAPES)
def test_draws(cuda, rows, V, mode, dtype):
    if rows * V > 10 ** 6 and dtype == "f16":
        pytest.skip("covered in bf16")
    rng = np.random.default_rng(rows + V)
    x = (3 * rng.standard_normal((rows, V))).astype(np.float32)
    if V > 100:
        x[:, ::7][rng.random((rows, x[:, ::7].shape[1])) < 0.1] = -np.inf
    check(cuda, cu(x, dtype), rng.random(rows).astype(np.float32), what=mode, **settings(rng, rows, mode))


@pytest.mark.parametrize("V", [7, 33, 1025, 6000, 40000])
def test_ties(cuda, V):
    """Few distinct values: every cut falls among equals, index order decides."""
    rng = np.random.default_rng(V)
    rows = 60
    x = rng.integers(-3, 3, (rows, V)).astype(np.float32)
    x[:10] = 2.0                      # all equal
    x[10:20] = np.float32(-3.4028235e38)   # the lowest value everywhere
    x[20:24, 1:] = np.float32(-3.4028235e38)
    x[24:28] *= -0.0                  # zeros of both signs
    u = rng.random(rows).astype(np.float32)
    k = rng.integers(1, V + 1, rows)
    p = rng.uniform(0.01, 0.999, rows)
    p[:3] = (0.5, 0.25, 0.75)
    ones = np.ones(rows)
    check(cuda, cu(x), u, k=k, what="top-k")
    check(cuda, cu(x), u, p=p, what="top-p")
    check(cuda, cu(x), u, k=k, p=p, what="both")
    check(cuda, cu(x), u, mp=ones, what="min-p 1")
    check(cuda, cu(x), u, T=0 * ones, what="greedy")
    check(cuda, cu(x), u, what="plain")


@pytest.mark.parametrize("V", [5, 1025, 70000])
def test_masked_rows(cuda, V):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((14, V)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, V - 1] = -1e30               # one entry left, the last
    x[3, 0] = np.nan
    x[4, ::2] = np.nan
    x[5, V // 2] = np.inf
    x[6, [0, V - 1]] = np.inf         # two infinite ones share everything
    x[7] = -3.4028235e38
    x[7, 3] = 0.0
    x[8] = np.where(np.arange(V) % 2, -np.inf, -3.4028235e38)
    x[9] = 3.4028235e38
    x[10, 0], x[10, 1] = 3.4028235e38, -3.4028235e38
    x[11] = -np.inf
    x[11, 2:4] = 1.0
    u = np.linspace(0.03, 0.97, 14).astype(np.float32)
    n = np.full(14, 3)
    half = np.full(14, 0.5)
    for kw in (dict(), dict(k=n), dict(p=half), dict(k=n, p=half), dict(mp=half * 0.1), dict(T=0 * half),
               dict(T=half, k=n, p=half, mp=half)):
        check(cuda, cu(x), u, what=str(sorted(kw)), **kw)


def test_extreme_settings(cuda):
    rng = np.random.default_rng(3)
    V = 1025
    x = np.tile((2 * rng.standard_normal((1, V))).astype(np.float32), (9, 1))
    u = rng.random(9).astype(np.float32)
    T = np.array([0.0, -1.0, np.nan, np.inf, 1e-30, 1e30, 1e-45, 3.0, 1e-3], np.float32)
    check(cuda, cu(x), u, T=T, what="temperatures")
    check(cuda, cu(x), u, k=np.array([1, V, V + 5, 0, -1, V - 1, 2, 2 ** 31 - 1, 500]), what="top_k")
    check(cuda, cu(x), u, p=np.array([0.0, -1.0, 1e-9, 0.9999999, 1.0, 1.5, np.nan, np.inf, 0.5]), what="top_p")
    check(cuda, cu(x), u, mp=np.array([0.0, -1.0, 1e-9, 1.0, 2.0, np.nan, np.inf, 0.999, 0.5]), what="min_p")
    edge = np.array([0.0, -1.0, np.nan, 1.0, 2.0, np.inf, 1 - 2.0 ** -24, 2.0 ** -40, 0.5], np.float32)
    check(cuda, cu(x), edge, k=np.full(9, 50), what="u")
    # scales of the logits that the bins do not fit
    for s in (1e-6, 1e4, 1e30):
        check(cuda, cu((x * s).astype(np.float32)), u, k=np.full(9, 40), p=np.full(9, 0.9), T=np.full(9, s), what=f"scale {s}")


@pytest.mark.parametrize("rows,V", [(5, 1000), (2, 40000)])
def test_pitch_offset_and_no_logprobs(cuda, rows, V):
    import torch
    rng = np.random.default_rng(1)
    wide = cu(rng.standard_normal((rows, V + 9)).astype(np.float32), "bf16", 1)
    u = rng.random(rows).astype(np.float32)
    tok, _ = check(cuda, wide[:, 4:4 + V], u, p=np.full(rows, 0.8))
    t2 = empty(rows, torch.int32)
    cuda.sample_rows(wide[:, 4:4 + V], cu(u), t2, top_p=cu(np.full(rows, 0.8, np.float32)))
    assert torch.equal(tok, t2)


def test_repeats_streams_graph(cuda):
    import torch
    rng = np.random.default_rng(2)
    for rows, V in ((64, 1025), (3, 50000)):
        x = cu((3 * rng.standard_normal((rows, V))).astype(np.float32))
        u, p = cu(rng.random(rows).astype(np.float32)), cu(np.full(rows, 0.9, np.float32))
        want, wl = empty(rows, torch.int32), empty(rows)
        cuda.sample_rows(x, u, want, wl, top_p=p)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = [(empty(rows, torch.int32), empty(rows)) for _ in range(8)]
        for i, (t, l) in enumerate(outs):
            cuda.sample_rows(x, u, t, l, top_p=p, stream=streams[i & 1])
        torch.cuda.synchronize()
        assert all(torch.equal(t, want) and torch.equal(l, wl) for t, l in outs)
        y = torch.zeros_like(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cuda.sample_rows(y, u, outs[0][0], outs[0][1], top_p=p)
        y.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0][0], want) and torch.equal(outs[0][1], wl)


def test_greedy_is_the_argmax(cuda):
    """With T = 0 the tokens are pkcu_argmax_rows's."""
    import torch
    rng = np.random.default_rng(4)
    x = cu(rng.integers(0, 50, (500, 1025)).astype(np.float32))
    a, t = empty(500, torch.int32), empty(500, torch.int32)
    cuda.call("pkcu_argmax_rows", x.data_ptr(), a.data_ptr(), 500, 1025, cuda.stream_handle())
    cuda.sample_rows(x, torch.rand(500, device="cuda"), t, temperature=torch.zeros(500, device="cuda"))
    assert torch.equal(a, t)


@pytest.mark.parametrize("dtype,V", [("f32", 5), ("f32", 1027), ("bf16", 9), ("bf16", 1030), ("bf16", 2016), ("f16", 2017),
                                     ("bf16", 40001)])
def test_rows_of_every_alignment(cuda, dtype, V):
    """A pitch of one entry more than a multiple of 16 bytes: rows start at every
    place that their type allows; enough of them for a warp per row where V allows."""
    rng = np.random.default_rng(V)
    rows = 1500 if V < 5000 else 20
    pitch = (V + 7) // 8 * 8 + 1
    wide = cu((3 * rng.standard_normal((rows, pitch))).astype(np.float32), dtype, 1)
    wide[:, V:] = 50.0   # never a row's
    check(cuda, wide[:, :V], rng.random(rows).astype(np.float32), **settings(rng, rows, "mixed"))


@pytest.mark.parametrize("rows,V", [(6, 32000), (2, 131072), (160, 20000)])
def test_wide_nuclei(cuda, rows, V):
    """Nuclei of most of the row, whose entries weigh little each; after a top-k too."""
    rng = np.random.default_rng(V)
    x = (2.5 * rng.standard_normal((rows, V))).astype(np.float32)
    x[::2, rng.integers(0, V, 4)] += 9.0
    u = rng.random(rows).astype(np.float32)
    p = np.resize(np.array([0.9, 0.97, 0.99, 0.999, 0.9999, 0.5], np.float32), rows)
    for dtype in ("f32", "bf16"):
        check(cuda, cu(x, dtype), u, p=p, T=np.full(rows, 1.1), what="top-p")
        check(cuda, cu(x, dtype), u, p=p, k=np.full(rows, V // 3), what="both")
