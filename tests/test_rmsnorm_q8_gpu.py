"""GPU: pkcu_residual_rms_norm_q8 against its formula in 64 bits.

Tolerances. x_out: y + bias and the multiply-add round once each in fp32, the
result once to the stream's type. scale: the sum of squares of D entries in
fp32, each thread of at least 32 per row adding ceil(D / 32) of them and five
to ten levels joining the threads, is off by at most (ceil(D / 32) + 12) 2^-24
relative (half of that after the square root); the products and quotients
around it round at most six more times. q: t, max|t|, Q / max|t| and their
product round once each (4 x 2^-24 relative), then the rounding to 8 bits is
off by half a step: 1/2 (int8); 2^-4 relative, or 2^-10 below 2^-6 (e4m3)."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import HALF_STEP, cu, f64, rms_q8, torch_dtype

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


def run(cuda, x, y, bias, alpha, gamma, q, pitch=None, x_out=None, **kw):
    import torch
    rows, D = x.shape
    pitch = pitch or D
    qt = empty((rows, pitch), torch.uint8).fill_(0x55).view(torch_dtype(q))
    scales = empty(rows).fill_(-1.0)
    if x_out is None and y is not None:
        x_out = empty(x.shape, x.dtype)
    cuda.residual_rms_norm_q8(x, y, bias, alpha, gamma, EPS, x_out, qt, scales, **kw)
    return x_out, qt, scales


def check(x_stored, gamma, q_got, scales, q, rows=None):
    """q and scales against the norm of the stored rows."""
    D = x_stored.shape[1]
    Q = 127.0 if q == "i8" else 448.0
    want_s, v = rms_q8(x_stored, gamma, EPS, Q)
    tol = ((-(-D // 32) + 12) / 2 + 6) * U
    assert (np.abs(scales - want_s) <= tol * want_s).all(), np.max(np.abs(scales - want_s) / want_s) / tol
    err = np.abs(q_got - v)
    if q == "i8":
        bad = err > 0.5 + 127 * 4 * U
    else:
        bad = err > np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10) * (1 + 64 * U)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3])


SHAPES = [(1, 1024), (7, 1024), (375, 1024), (3000, 1024), (1, 1), (5, 3), (2, 31), (33, 32), (9, 100), (1300, 130),
          (2, 640), (3, 1025), (4, 4096), (301, 4100), (2, 8192), (3, 8200), (1, 33000), (2, 65536)]


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", SHAPES)
def test_matches_formula(cuda, rows, D, dtype, q):
    r = np.random.default_rng(rows * 7 + D)
    x = cu(2 * r.standard_normal((rows, D)).astype(np.float32), dtype)
    y = cu(r.standard_normal((rows, D)).astype(np.float32), dtype)
    bias = r.standard_normal(D).astype(np.float32)
    gamma = (1 + 0.3 * r.standard_normal(D)).astype(np.float32)
    pitch = D + 5
    for alpha, b in ((0.5, bias), (1.0, None)):
        x_out, qt, scales = run(cuda, x, y, None if b is None else cu(b), alpha, cu(gamma), q, pitch)
        xo = f64(x_out)
        add = f64(y) + (0 if b is None else b.astype(np.float64))
        want = f64(x) + alpha * add
        tol = HALF_STEP[dtype] * np.abs(want) + 2 * U * (np.abs(f64(x)) + np.abs(add))
        if dtype == "f16":
            tol += 2.0 ** -25   # half a step of a subnormal
        assert (np.abs(xo - want) <= tol * (1 + 2.0 ** -7)).all()
        check(xo, gamma, f64(qt)[:, :D], f64(scales), q)
        import torch
        assert (qt.view(torch.uint8)[:, D:] == 0x55).all()   # the padding columns are left
    # without y: the norm of x, and the same as a fused call's second half
    _, qt2, scales2 = run(cuda, x_out, None, None, 0.0, cu(gamma), q, pitch)
    assert (qt2.view(torch.uint8) == qt.view(torch.uint8)).all() and (scales2 == scales).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1024, 1000, 72])
def test_in_place_and_misaligned(cuda, dtype, D):
    import torch
    r = np.random.default_rng(D)
    xs, ys = (r.standard_normal((13, D)).astype(np.float32) for _ in range(2))
    g, b = (r.standard_normal(D).astype(np.float32) for _ in range(2))
    want = run(cuda, cu(xs, dtype), cu(ys, dtype), cu(b), 0.5, cu(g), "i8")
    x = cu(xs, dtype)
    got = run(cuda, x, cu(ys, dtype), cu(b), 0.5, cu(g), "i8", x_out=x)
    for w, h in zip(want, got):
        assert torch.equal(w, h)
    for off in (1, 2, 3):   # starts that are aligned to their type alone
        got = run(cuda, cu(xs, dtype, off), cu(ys, dtype, off), cu(b, None, off), 0.5, cu(g, None, off), "i8",
                  x_out=cu(np.zeros_like(xs), dtype, off))
        assert torch.equal(got[0], want[0])
        # another kernel sums the squares in another order: within the bound of either
        check(f64(got[0]), g, f64(got[1]), f64(got[2]), "i8")


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("D", [1024, 1001])
def test_special_rows(cuda, D, q):
    r = np.random.default_rng(5)
    x = r.standard_normal((10, D)).astype(np.float32)
    x[0] = 0.0
    x[1, 3] = np.nan
    x[2, D - 1] = np.inf
    x[3, 0] = -np.inf
    x[4] *= 1e-36       # the largest entry's reciprocal times Q overflows
    x[5] *= 1e17
    x[6] = 0.0
    x[6, 17] = -2.5     # one entry
    x[7] = 1.0          # all the same
    x[8] *= 1e-12
    gamma = np.ones(D, np.float32)
    gamma[5] = -2.0
    gamma[6] = 0.0
    _, qt, s = run(cuda, cu(x), None, None, 0.0, cu(gamma), q)
    s, qv = f64(s), f64(qt)
    assert s[0] == 0 and (qv[0] == 0).all()
    for i in (1, 2, 3):
        assert np.isnan(s[i]) and (qv[i] == 0).all()
    rows = [4, 5, 6, 7, 8, 9]
    check(x[rows], gamma, qv[rows], s[rows], q)
    # gamma zero everywhere: a row of zeros
    _, qt, s = run(cuda, cu(x[9:]), None, None, 0.0, cu(np.zeros(D, np.float32)), q)
    assert f64(s)[0] == 0 and (f64(qt) == 0).all()
    # a NaN in gamma reaches every row
    gamma[1] = np.nan
    _, qt, s = run(cuda, cu(x[9:]), None, None, 0.0, cu(gamma), q)
    assert np.isnan(f64(s)[0]) and (f64(qt) == 0).all()


def test_stream_and_graph(cuda):
    import torch
    r = np.random.default_rng(1)
    x, y = (cu(r.standard_normal((375, 1024)).astype(np.float32)) for _ in range(2))
    g = cu(np.ones(1024, np.float32))
    want = run(cuda, x, y, None, 1.0, g, "e4m3")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [empty((375, 1024)), empty((375, 1024), torch.uint8).view(torch.float8_e4m3fn), empty(375)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cuda.residual_rms_norm_q8(x, y, None, 1.0, g, EPS, *got)
    x.mul_(2.0)
    y.mul_(2.0)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], 2 * want[0])
    check(f64(got[0]), np.ones(1024), f64(got[1]), f64(got[2]), "e4m3")
    out = run(cuda, x, y, None, 1.0, g, "e4m3", stream=side)
    side.synchronize()
    assert torch.equal(out[0], got[0]) and torch.equal(out[2], got[2])


def test_no_rows(cuda):
    cuda.call("pkcu_residual_rms_norm_q8", None, None, None, 1.0, None, EPS, 0, None, None, 1, 1024, None, 0, 1024,
              None)


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("rows,D,dtype,parts", [(1184, 4104, "bf16", "yb"), (1185, 8192, "f16", "y"), (2400, 5000, "bf16", ""),
                                                (1700, 8184, "bf16", "y"), (1300, 8192, "f32", "yb")])
def test_many_wide_rows(cuda, rows, D, dtype, parts, q):
    """In place, rows of NaN, of infinity and of zeros among the others, what
    lies behind a row left as it was; twice the same bits, and from a graph."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows + D)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = (2 * n(rows, D)).to(torch_dtype(dtype))
    x[5], x[rows - 1] = 0.0, 0.0
    x[7, D - 1], x[rows - 2, 0], x[9] = float("nan"), float("inf"), 1e-4
    y = n(rows, D).to(x.dtype) if parts else None
    if parts:
        y[5], y[rows - 1] = 0.0, 0.0
    bias = 0.1 * n(D) if "b" in parts else None
    gamma = 1 + 0.2 * n(D)
    outs = []
    for _ in range(2):
        xo = x.clone()
        outs.append(run(cuda, xo, y, bias, 0.5, gamma, q, pitch=D + 16 - D % 8, x_out=xo if parts else None))
    xo, qt, scales = outs[0]
    view = lambda t: t.view(torch.uint8)
    assert torch.equal(view(qt), view(outs[1][1])) and torch.equal(scales.view(torch.int32), outs[1][2].view(torch.int32))
    stored = xo if parts else x
    if parts:
        add = y.double() if bias is None else y.double() + bias.double()
        want = x.double() + 0.5 * add
        tol = HALF_STEP[dtype] * want.abs() + 2 * U * (want.abs() + x.double().abs()) + 2.0 ** -25 * (dtype == "f16")
        fine = torch.isfinite(want)
        assert ((stored.double() - want).abs()[fine] <= tol[fine]).all()
    odd = ~torch.isfinite(stored.double()).all(dim=1)
    assert odd.nonzero().flatten().tolist() == [7, rows - 2]
    s = f64(scales)
    assert np.isnan(s[[7, rows - 2]]).all() and (view(qt)[[7, rows - 2], :D] == 0).all()
    if bias is None:
        assert s[5] == 0 and s[rows - 1] == 0 and (view(qt)[5, :D] == 0).all()
    assert (view(qt)[:, D:] == 0x55).all()
    # rows of all parts of the run, among them the last of every group
    some = sorted(({0, 1, 5, 9, rows - 1, rows - 3} | set(range(11, rows, 37)) | set(range(rows - 300, rows - 2, 7))) - {7})
    if bias is None:
        some = [i for i in some if i not in (5, rows - 1)]
    check(f64(stored[some]), f64(gamma), f64(qt[some][:, :D].float()), s[some], q)
    q2, s2 = empty(qt.shape, torch.uint8).fill_(0x55).view(qt.dtype), empty(rows)
    xi, xg = torch.zeros_like(x), torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.residual_rms_norm_q8(xi, y, bias, 0.5, gamma, EPS, xg if parts else None, q2, s2)
    xi.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(view(q2), view(qt)) and torch.equal(s2.view(torch.int32), scales.view(torch.int32))


@pytest.mark.parametrize("D,offset", [(9001, 0), (16384, 0), (16384, 1), (20008, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_rows_in_place(cuda, dtype, D, offset):
    r = np.random.default_rng(D)
    x, y = (cu(r.standard_normal((5, D)).astype(np.float32), dtype, offset) for _ in range(2))
    gamma = cu((1 + 0.2 * r.standard_normal(D)).astype(np.float32))
    before = f64(x)
    run(cuda, x, y, None, 1.0, gamma, "i8", x_out=x)
    want = before + f64(y)
    assert (np.abs(f64(x) - want) <= (HALF_STEP[dtype] + 2 * U) * np.abs(want) + U * np.abs(before)).all()
    x, q, s = x, *run(cuda, x, None, None, 0.0, gamma, "e4m3")[1:]
    check(f64(x), f64(gamma), f64(q), f64(s), "e4m3")
