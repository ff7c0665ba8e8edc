"""GPU: pkcu_wmatmul_q8's activations over the whole range of their argument, from
the smallest kernel (one token) and from the CTA pairs (2500 tokens).

The products are 0 and the bias is the argument v, exactly. Values of +-2^-40 ..
+-3.4e38 and +-infinity; in all three output types.

Tolerance: 16 x 2^-24 of the value, as where the activations are tested at +-10^1
.. 10^38; what goes to 0 is within 1e-30 of it; the output type rounds once, by
half a step (fp16 also by half a subnormal step, 2^-25), and to infinity from half
a step above its largest value on: 65504 + 16 in fp16; (2 - 2^-7) 2^127 + 2^119 =
(2 - 2^-8) 2^127 in bf16, which fp32's largest value lies above."""
import math

import numpy as np
import pytest

from gpuhelp import empty
from q8help import HALF_STEP, cu, f64, torch_dtype

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N = 1024


def arguments():
    big = np.array([1e30, 1e38, 2.3e38, 2.36e38, 2.4e38, 3e38, 3.4028235e38, math.inf])
    some = np.array([0.0, 2.0 ** -40, 1e-3, 0.5, 1.0, 5.0, 17.0, 85.9, 86.0, 86.1, 87.0, 88.5, 100.0, 199.0, 201.0, 1e3, 65504.0, 7e4, 1e6])
    v = np.concatenate([big, some, -big, -some]).astype(np.float32)
    return np.resize(v, N)


def values(cuda, M, out, act, v):
    """The activation of v by the kernel that M tokens take, every token alike."""
    import torch
    w, a = torch.zeros(16, N, dtype=torch.int8, device="cuda"), torch.zeros(M, 16, dtype=torch.int8, device="cuda")
    with cuda.WeightQ8(w, 1.0) as W:
        c = empty((M, N), torch_dtype(out))
        cuda.wmatmul_q8(a, cu(np.ones(M, np.float32)), W, c, bias=cu(v), act=act)
    bits = c.view({"f32": torch.int32}.get(out, torch.int16))
    assert torch.equal(bits, bits[:1].expand(M, N))
    return f64(c[0])


def compare(got, want, tol, out):
    if out != "f32":
        border = 65520.0 if out == "f16" else (2 - 2.0 ** -8) * 2.0 ** 127
        want = np.where(np.abs(want) >= border, np.copysign(math.inf, want), want)
    if out == "f16":
        tol = tol + 2.0 ** -25
    same = got == want   # the infinite ones
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= tol + HALF_STEP[out] * np.abs(want) * (1 + 2.0 ** -7)
    bad = np.flatnonzero(~(same | near))
    assert not len(bad), [(i, got[i], want[i]) for i in bad[:5]]


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", [None, "relu", "swish", "tanh"])
@pytest.mark.parametrize("M", [1, 200, 2500])
def test_whole_range(cuda, M, act, out):
    v = arguments()
    x = v.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        want = {None: x, "relu": np.maximum(x, 0), "tanh": np.tanh(x),
                "swish": np.where(x < -700, 0.0, x / (1 + np.exp(-np.maximum(x, -700))))}[act]
    fin = np.where(np.isinf(want), 0, np.abs(want))
    compare(values(cuda, M, out, act, v), want, 16 * U * fin + 1e-30, out)


@pytest.mark.parametrize("act", [None, "relu", "swish", "gelu", "tanh"])
@pytest.mark.parametrize("M", [1, 2500])
def test_nan_stays(cuda, M, act):
    v = np.full(N, math.nan, np.float32)
    assert np.isnan(values(cuda, M, "f32", act, v)).all()


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M", [1, 200, 2500])
def test_gelu(cuda, M, out):
    """The GELU's small values left of 0 have the relative error of the others.
    g = |v| e^(-v^2 / 2) P: the exponent s = a^2 (log2 e) / 2 has three roundings (a^2,
    the constant, their product), v^2 / 2 x 3 x 2^-24 of the power, whose approximation
    is off by 2^-22; t = 1 / (1 + 0.3 |v|) by 3 x 2^-24 (the sum, the reciprocal's unit
    in the last place), which P multiplies by |t P' / P| <= 2.7; P by its distance, 1,
    and its steps, 4; two products round: (1.5 v^2 + 4 + 8.1 + 5 + 2) 2^-24 < (2 v^2 +
    20) 2^-24, and the difference max(v, 0) - g once more where it is not exact. Where
    the power is below fp32's normal numbers (|v| > 13.2) the value is below 1e-36."""
    from scipy.special import erfc
    v = np.concatenate([arguments()[:54], np.linspace(-14, -2, 601), np.linspace(-2, 9, 300)]).astype(np.float32)
    v = np.resize(v, N)
    x = v.astype(np.float64)
    with np.errstate(invalid="ignore"):
        want = np.where(x < -30, 0.0, 0.5 * x * erfc(-x / math.sqrt(2)))
    fin = np.where(np.isinf(want), 0, np.abs(want))
    compare(values(cuda, M, out, "gelu", v), want, (2 * np.minimum(x * x, 1e4) + 20) * U * fin + 1e-36, out)
