"""GPU: pkcu_sample_rows' log-probabilities are the definition's, rounded once.

In fp64 the exponent is off by 4 x 2^-53 of its value (at most 60 here) and the
logarithm by 4 x 10^-13 and as much as the sum: 2 x 10^-13 of it, and 2^-45 of the
largest weight per entry at most, for these rows 2.1 x 10^-12 together (computed from
them); the result rounds to fp32 by 2^-24 of its value."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu, f64
from test_sample_rows_gpu import U, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k,p", [(0, 1.0), (50, 1.0), (0, 0.9)])
@pytest.mark.parametrize("rows,V", [(1500, 100), (1200, 1025), (300, 1025), (64, 32000), (8, 131072)])
def test_rounded_once(cuda, rows, V, k, p, dtype):
    import torch
    rng = np.random.default_rng(rows + V)
    x = cu((2.5 * rng.standard_normal((rows, V))).astype(np.float32), dtype)
    u, T = rng.random(rows).astype(np.float32), rng.uniform(0.6, 1.4, rows).astype(np.float32)
    tok, lp = empty(rows, torch.int32), empty(rows)
    kd = cu(np.full(rows, k, np.int32)) if k else None
    pd = cu(np.full(rows, p, np.float32)) if p < 1 else None
    cuda.sample_rows(x, cu(u), tok, lp, temperature=cu(T), top_k=kd, top_p=pd)
    got, t, host = f64(lp), f64(tok), f64(x)
    for i in range(rows):
        want = plain(host[i], float(u[i]), float(T[i]), k, float(np.float32(p)), 0.0)
        assert t[i] == want[0]
        assert abs(got[i] - want[1]) <= U * abs(want[1]) * (1 + 2.0 ** -7) + 1e-11, (i, got[i], want[1])
