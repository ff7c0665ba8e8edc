"""GPU: pkcu_wmatmul_q8 against its formula in 64 bits.

Tolerance. An int8 sum is exact; the conversion, the two scales and the bias
round once each in fp32: |v - v64| <= 3 U |P| + U |v| =: e with P the product's
part of v and U = 2^-24. An e4m3 sum is made by MMAs of 32 products; each adds
at most 2^-22 of the magnitudes met so far, together (K / 32 + 1) 2^-22 times
sum |a w| (times the scales). The activations have slopes of at most 1.13 and
are off by a few fp32 steps: 8 U of their value, for the GELU 4 U of v (1 + erf
cancels). The residual's multiply-add rounds once more, C's type once."""
import math

import numpy as np
import pytest

from gpuhelp import empty
from q8help import HALF_STEP, cu, f64, torch_dtype

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def operands(rng, M, K, N, q, col_scales=True):
    if q == "i8":
        a, w = (rng.integers(-128, 128, s).astype(np.int8) for s in ((M, K), (K, N)))
        a, w = cu(a), cu(w)
    else:
        a, w = (cu(np.clip(100 * rng.standard_normal(s), -448, 448).astype(np.float32), "e4m3") for s in ((M, K), (K, N)))
    lim = 127.0 if q == "i8" else 100.0
    sa = (rng.uniform(0.5, 2, M) / lim).astype(np.float32)
    sw = (rng.uniform(0.5, 2, N if col_scales else 1) / lim / math.sqrt(K)).astype(np.float32)
    return a, w, sa, sw


def padded(a, fill=0x7f):
    """a [M, K] with a pitch that is a multiple of 16; the padding holds NaN (e4m3) or 127."""
    import torch
    M, K = a.shape
    p = torch.full((M, (K + 15) // 16 * 16 + 16), fill, dtype=torch.uint8, device="cuda").view(a.dtype)
    p[:, :K] = a
    return p


def erf64(x):
    import torch
    return torch.erf(torch.from_numpy(np.ascontiguousarray(x))).numpy()


def want_and_tol(a, w, sa, sw, bias, act, r, rs, out, q):
    A, W = f64(a), f64(w)
    K = A.shape[1]
    P = (A @ W) * sa.astype(np.float64)[:, None] * sw.astype(np.float64)[None, :]
    v = P + (0 if bias is None else bias.astype(np.float64))
    e = 3 * U * np.abs(P) + U * np.abs(v)
    if q == "e4m3":
        mag = (np.abs(A) @ np.abs(W)) * sa.astype(np.float64)[:, None] * sw.astype(np.float64)[None, :]
        e = e + (K / 32 + 1) * 2.0 ** -22 * mag
    with np.errstate(over="ignore"):
        f = {None: lambda t: t, "relu": lambda t: np.maximum(t, 0), "swish": lambda t: t / (1 + np.exp(-t)),
             "tanh": np.tanh, "gelu": lambda t: 0.5 * t * (1 + erf64(t / math.sqrt(2)))}[act](v)
    ef = 1.13 * e + (8 * U * np.abs(f) if act in ("swish", "tanh") else 4 * U * np.abs(v) if act == "gelu" else 0)
    o = rs * f + (0 if r is None else f64(r))
    tol = abs(rs) * ef + 2 * U * (np.abs(o) + np.abs(rs * f)) + HALF_STEP[out] * np.abs(o) + 1e-30
    if out == "f16":
        tol = tol + 2.0 ** -25
    return o, tol * (1 + 2.0 ** -7)


def check(got, want, tol, what=""):
    err = np.abs(got - want)
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{bad.size} outside; first at {np.argwhere(bad)[0]}; "
                           f"max err/tol {np.nanmax(err / tol):.3f}")


SHAPES = [(1, 1024, 4096), (1, 1, 1), (2, 15, 7), (3, 16, 32), (5, 31, 127), (16, 64, 128), (17, 127, 129),
          (32, 640, 1025), (33, 128, 640), (64, 129, 33), (65, 1000, 1025), (129, 640, 640), (200, 1024, 1024),
          (257, 100, 300), (300, 1024, 4096), (1000, 4096, 1024), (2500, 1024, 2048), (1, 8192, 128), (128, 2048, 256)]


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product(cuda, M, K, N, q):
    rng = np.random.default_rng(M * 31 + K * 7 + N)
    a, w, sa, sw = operands(rng, M, K, N, q)
    bias = rng.standard_normal(N).astype(np.float32)
    ap = padded(a)
    with cuda.WeightQ8(w, cu(sw)) as W:
        for out, act, b, res, rs in (("f32", None, None, False, 1.0), ("bf16", "swish", bias, False, 1.0),
                                     ("f32", None, bias, True, 0.5), ("f16", "relu", bias, True, 1.0)):
            r = cu(rng.standard_normal((M, N)).astype(np.float32), out) if res else None
            c = empty((M, N), torch_dtype(out)).fill_(math.nan)
            cuda.wmatmul_q8(ap, cu(sa), W, c, bias=None if b is None else cu(b), act=act, residual=r, rscale=rs)
            check(f64(c), *want_and_tol(a, w, sa, sw, b, act, r, rs, out, q), what=f"{out} {act}")


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", [None, "relu", "swish", "gelu", "tanh"])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_epilogues(cuda, M, act, out):
    K, N = 256, 1030
    rng = np.random.default_rng(M)
    a, w, sa, sw = operands(rng, M, K, N, "i8", col_scales=False)
    bias = (4 * rng.standard_normal(N)).astype(np.float32)
    r = cu(rng.standard_normal((M, N)).astype(np.float32), out)
    with cuda.WeightQ8(w, cu(sw)) as W:
        for b, res, rs in ((bias, r, 0.5), (None, r, -1.0), (bias, None, 2.0)):
            c = empty((M, N), torch_dtype(out))
            cuda.wmatmul_q8(a, cu(sa), W, c, bias=None if b is None else cu(b), act=act, residual=res, rscale=rs)
            check(f64(c), *want_and_tol(a, w, sa, sw, b, act, res, rs, out, "i8"))


@pytest.mark.parametrize("M", [3, 150, 700])
def test_pitches_in_place_and_what_lies_around(cuda, M):
    """Rows of C, R and A inside wider ones, starts aligned to their type alone,
    C in place of R; nothing beside the rows is written."""
    import torch
    K, N = 200, 333
    rng = np.random.default_rng(M)
    a, w, sa, sw = operands(rng, M, K, N, "i8")
    bias = rng.standard_normal(N).astype(np.float32)
    wide = cu(rng.standard_normal((M + 2, N + 10)).astype(np.float32), None, 1)
    before = wide.clone()
    x = wide[1:M + 1, 3:3 + N]
    r = x.clone()
    with cuda.WeightQ8(w, cu(sw)) as W:
        cuda.wmatmul_q8(padded(a), cu(sa), W, x, bias=cu(bias), act="swish", residual=x, rscale=0.5)
    check(f64(x), *want_and_tol(a, w, sa, sw, bias, "swish", r, 0.5, "f32", "i8"))
    before[1:M + 1, 3:3 + N] = x
    assert torch.equal(wide, before)


def test_largest_int8_sums(cuda):
    import torch
    K = 131071
    w = torch.full((K, 5), -128, dtype=torch.int8, device="cuda")
    a = torch.full((2, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    c = empty((2, 5))
    with cuda.WeightQ8(w, 1.0) as W:
        cuda.wmatmul_q8(a, one, W, c)
    assert (f64(c) == np.float32(16384 * K)).all()


def test_rows_of_nan_and_zero_scales(cuda):
    rng = np.random.default_rng(0)
    a, w, sa, sw = operands(rng, 20, 64, 40, "i8")
    sa[3] = 0.0
    sa[5] = np.nan
    with cuda.WeightQ8(w, cu(sw)) as W:
        for act in (None, "relu", "swish", "gelu", "tanh"):
            c = empty((20, 40))
            cuda.wmatmul_q8(a, cu(sa), W, c, act=act)
            got = f64(c)
            assert (got[3] == 0).all() and np.isnan(got[5]).all() and np.isfinite(np.delete(got, 5, 0)).all()


def test_streams_graph_and_repeats(cuda):
    """The same bits from run to run, from two streams at once and from a
    replayed graph that reads new inputs."""
    import torch
    rng = np.random.default_rng(9)
    for M in (1, 48, 600):
        a, w, sa, sw = operands(rng, M, 1024, 1025, "e4m3")
        sad = cu(sa)
        with cuda.WeightQ8(w, cu(sw)) as W:
            want = empty((M, 1025))
            cuda.wmatmul_q8(a, sad, W, want, act="swish")
            torch.cuda.synchronize()
            s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
            outs = [empty((M, 1025)) for _ in range(6)]
            for i, o in enumerate(outs):
                cuda.wmatmul_q8(a, sad, W, o, act="swish", stream=(s1, s2)[i & 1])
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in outs)
            b = a.clone()
            b.view(torch.uint8).zero_()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                cuda.wmatmul_q8(b, sad, W, outs[0], act="swish")
            b.copy_(a)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want)


def test_no_rows(cuda):
    import torch
    w = torch.zeros(64, 8, dtype=torch.int8, device="cuda")
    with cuda.WeightQ8(w, 1.0) as W:
        cuda.wmatmul_q8(torch.zeros(0, 64, dtype=torch.int8, device="cuda"), torch.zeros(0, device="cuda"), W,
                        torch.zeros(0, 8, device="cuda"))
        with pytest.raises(cuda.PkCudaError, match="activation"):
            cuda.call("pkcu_wmatmul_q8", 4096, 64, 4096, W.handle, None, 5, None, 0, 1.0, 4096, 8, 0, 4, None)
        for change, word in ((dict(lda=63), "pitch"), (dict(lda=48), "pitch"), (dict(a=4104), "16-byte"),
                             (dict(ldc=7), "shorter"), (dict(dtype=1), "type"), (dict(M=-1), "rows"),
                             (dict(c=None), "NULL"), (dict(sa=None), "NULL"), (dict(c=4097), "aligned"),
                             (dict(r=4096, ldr=7), "shorter"), (dict(r=4098, ldr=8), "aligned"),
                             (dict(bias=4097), "aligned")):
            p = dict(a=4096, lda=64, sa=4096, w=W.handle, bias=None, act=2, r=None, ldr=0, rs=1.0, c=4096, ldc=8,
                     dtype=0, M=4)
            p.update(change)
            with pytest.raises(cuda.PkCudaError, match=word):
                cuda.call("pkcu_wmatmul_q8", *p.values(), None)
