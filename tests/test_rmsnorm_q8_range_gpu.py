"""GPU: pkcu_residual_rms_norm_q8 at the ends of its range. A row whose sum of squares
or whose product of an entry and its gamma passes fp32 has q = 0 and scale NaN, as
the header says, in every kernel (a warp, a CTA, a ring of copies, rows above 8192),
and its neighbours what the formula gives; where only the norm passes fp32 and its
scale does not, so has the row itself.

Tolerances: those of the ordinary rows (the head of test_rmsnorm_q8_gpu.py); the scale
by r / Q has no more roundings than the other way."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu, f64, torch_dtype
from test_rmsnorm_q8_gpu import EPS, check

pytestmark = pytest.mark.gpu


def run(cuda, x, gamma, q):
    import torch
    rows, D = x.shape
    qt, s = empty((rows, (D + 15) // 16 * 16), torch.uint8).fill_(0x55).view(torch_dtype(q)), empty(rows)
    cuda.residual_rms_norm_q8(x, None, None, 0.0, gamma, EPS, None, qt, s)
    assert (qt.view(torch.uint8)[:, D:] == 0x55).all()
    return f64(qt)[:, :D], f64(s)


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(12, 200), (12, 203), (12, 512), (12, 1024), (12, 1001), (12, 2048), (12, 4096), (12, 8192),
                                    (1300, 8192), (12, 20000), (12, 9001)])
def test_rows_past_fp32(cuda, rows, D, dtype, q):
    import torch
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(rows, D, device="cuda", generator=g).clamp_(-3, 3)
    x[0] *= 1e25                    # squares
    x[1, D // 2] = 3e38             # one square
    x[3, 0] = -1e20                 # one square, and the product with a large gamma
    x[5] *= 1e17                    # inside the range, but for the product
    x[rows - 1] *= 1e30
    x = x.to(torch_dtype(dtype))
    gamma = 1 + 0.2 * torch.randn(D, device="cuda", generator=g)
    lost = [0, 1, 3, rows - 1]
    for gm, out in ((gamma, lost), (gamma * 1e25, lost + [5])):
        qv, s = run(cuda, x, gm, q)
        out = sorted(set(out))
        assert np.isnan(s[out]).all() and (qv[out] == 0).all()
        kept = [i for i in range(rows) if i not in out][:60]
        check(f64(x[kept]), f64(gm), qv[kept], s[kept], q)


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("D", [1024, 9000])
def test_a_norm_past_fp32_with_a_scale_that_is_not(cuda, q, D):
    x = np.zeros((2, D), np.float32)
    x[0, 3], x[1] = 0.5, 0.5
    gamma = np.full(D, 3e38, np.float32)
    qv, s = run(cuda, cu(x), cu(gamma), q)
    assert np.isfinite(s).all()
    check(x, gamma, qv, s, q)
