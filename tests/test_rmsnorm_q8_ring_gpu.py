"""GPU: pkcu_residual_rms_norm_q8 where many wide 16-bit rows go through rings of
bulk copies: numbers of rows at which the groups end at different places, on two
streams at once, the same bits every time and no wait that ran out (checked after
every test)."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import f64, torch_dtype
from test_rmsnorm_q8_gpu import EPS, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1184, 1185, 1331, 1332, 1333, 2369])
@pytest.mark.parametrize("D,dtype", [(4104, "f16"), (8192, "bf16")])
def test_rings_side_by_side(cuda, rows, D, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows * D)
    x, y = (torch.randn(rows, D, device="cuda", generator=g).to(torch_dtype(dtype)) for _ in range(2))
    gamma = 1 + 0.2 * torch.randn(D, device="cuda", generator=g)
    out = lambda: (empty((rows, D), x.dtype), empty((rows, D), torch.int8), empty(rows))
    want = out()
    cuda.residual_rms_norm_q8(x, y, None, 0.5, gamma, EPS, *want)
    some = sorted({0, 1, rows // 2, rows - 2, rows - 1})
    check(f64(want[0][some]), f64(gamma), f64(want[1][some]), f64(want[2][some]), "i8")
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [out() for _ in range(2)]
    for i in range(20):
        cuda.residual_rms_norm_q8(x, y, None, 0.5, gamma, EPS, *outs[i & 1], stream=streams[i & 1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))
    assert np.isfinite(f64(want[2])).all()
