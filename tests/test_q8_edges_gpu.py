"""GPU: the 8-bit operators where a program may come upon them unprepared: a
process whose first calls are captured, weights made on another stream, sums far
outside an activation's usual range, calls that the wrappers refuse."""
import os
import subprocess
import sys

import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu, f64

pytestmark = pytest.mark.gpu

FIRST_CALLS = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import pkcuda
torch.manual_seed(0)
x, y = torch.randn(ROWS, 1024, device="cuda"), torch.randn(ROWS, 1024, device="cuda")
g = torch.ones(1024, device="cuda")
q, s = torch.zeros(ROWS, 1024, dtype=torch.int8, device="cuda"), torch.zeros(ROWS, device="cuda")
W = pkcuda.WeightQ8(torch.randint(-127, 128, (1024, 1025), device="cuda").to(torch.int8), 1e-3)
logits = torch.zeros(ROWS, 1025, device="cuda")
u, p = torch.rand(ROWS, device="cuda"), torch.full((ROWS,), 0.9, device="cuda")
tok = torch.full((ROWS,), -5, dtype=torch.int32, device="cuda")
def run():
    pkcuda.residual_rms_norm_q8(x, y, None, 1.0, g, 1e-5, torch.empty_like(x), q, s)
    pkcuda.wmatmul_q8(q, s, W, logits)
    pkcuda.sample_rows(logits, u, tok, top_p=p)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run()
graph.replay()
torch.cuda.synchronize()
got = tok.clone(), logits.clone()
run()
torch.cuda.synchronize()
assert (tok >= 0).all() and torch.equal(tok, got[0]) and torch.equal(logits, got[1])
print("first calls captured")
"""


@pytest.mark.parametrize("rows", [1, 1000])
def test_first_calls_of_a_process_are_captured(cuda, rows):
    where = os.path.dirname(os.path.abspath(cuda.__file__))
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS.replace("ROWS", str(rows)), where], capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0 and "first calls captured" in out.stdout, out.stderr[-2000:]


def test_a_weight_made_on_another_stream(cuda):
    """A scale given as a number is there when the weight is made, whatever the
    current stream still has to do."""
    import torch
    data = cu(np.arange(64 * 8).reshape(64, 8).astype(np.float32) % 7, "i8")
    a, one = cu(np.ones((1, 64), np.float32), "i8"), cu(np.ones(1, np.float32))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)   # the current stream is busy for a tenth of a second
    with cuda.WeightQ8(data, 0.5, stream=side) as W:
        c = empty((1, 8))
        cuda.wmatmul_q8(a, one, W, c)
        assert (f64(c) == 0.5 * f64(data).sum(axis=0)).all()


@pytest.mark.parametrize("M", [1, 700])
@pytest.mark.parametrize("act", ["relu", "swish", "gelu", "tanh"])
def test_sums_far_outside(cuda, M, act):
    """Activations of +-10^1 .. 10^38: what goes to 0 is within 1e-30 of it, the
    rest within a few fp32 steps."""
    v = np.concatenate([s * 10.0 ** np.arange(1, 39) for s in (1, -1)])
    N = 256
    w = cu(np.ones((16, N), np.float32), "i8")
    sw = np.resize(v / 16, N).astype(np.float32)
    with cuda.WeightQ8(w, cu(sw)) as W:
        c = empty((M, N))
        cuda.wmatmul_q8(cu(np.ones((M, 16), np.float32), "i8"), cu(np.ones(M, np.float32)), W, c, act=act)
    x = 16.0 * sw.astype(np.float64)
    with np.errstate(over="ignore"):
        want = {"relu": np.maximum(x, 0), "swish": x / (1 + np.exp(-x)), "tanh": np.tanh(x),
                "gelu": np.where(x > 0, x, 0.0)}[act]
    tol = 16 * 2.0 ** -24 * np.abs(want) + 1e-30
    if act == "gelu":
        tol = tol + 4 * 2.0 ** -24 * 10.0 * (np.abs(x) < 20)   # the definition's value at -10 is -7e-23
    got = f64(c)
    assert (np.abs(got - want) <= tol).all(), np.argwhere(~(np.abs(got - want) <= tol))[:4]


def test_wrapper_refusals(cuda):
    import torch
    w = torch.zeros(64, 8, dtype=torch.int8, device="cuda")
    a, s, c = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(4, 8, device="cuda")
    W = cuda.WeightQ8(w, 1.0)
    for args, kw in (((a, s, W, c), dict(act="elu")), ((a, s[:3], W, c), {}), ((a.float(), s, W, c), {}),
                     ((a, s, W, c.t()), {}), ((a, s, W, c), dict(bias=s)), ((a, s, W, c), dict(residual=c.half())),
                     ((a, s.cpu(), W, c), {}), ((a, s, W, c.to(torch.int32)), {})):
        with pytest.raises(ValueError):
            cuda.wmatmul_q8(*args, **kw)
    W.close()
    with pytest.raises(ValueError, match="closed"):
        cuda.wmatmul_q8(a, s, W, c)
    x, g, q = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(4, 16, dtype=torch.int8, device="cuda")
    for change in (dict(x=x.t()), dict(y=x.half()), dict(gamma=g[:7]), dict(q=q[:3]), dict(q=q.t()), dict(x_out=x[:2]),
                   dict(scales=s[:2]), dict(x=x.double()), dict(x=x.cpu())):
        p = dict(x=x, y=x, bias=None, alpha=1.0, gamma=g, eps=1e-5, x_out=x, q=q, scales=s)
        p.update(change)
        with pytest.raises(ValueError):
            cuda.residual_rms_norm_q8(**p)
    u, t = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for args, kw in (((x[0], u, t), {}), ((x, u[:2], t), {}), ((x, u, t.long()), {}), ((x, u, t), dict(top_k=u)),
                     ((x, u, t), dict(top_p=t)), ((x.t(), u, t), {}), ((x.cpu(), u, t), {})):
        with pytest.raises(ValueError):
            cuda.sample_rows(*args, **kw)
