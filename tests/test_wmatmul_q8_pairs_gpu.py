"""GPU: pkcu_wmatmul_q8 for many tokens (CTA pairs), short kernels one after
another: a CTA of a pair leaves only when its partner's last signals have reached
it, so whatever takes its place on the SM (other pairs, one-CTA products, the norm)
finds its shared memory undisturbed. The same bits every time."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu, f64
from test_wmatmul_q8_gpu import check, operands, want_and_tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("M,K,N", [(2500, 16, 1024), (5000, 130, 512), (6000, 1024, 2048)])
def test_back_to_back(cuda, M, K, N, q):
    import torch
    rng = np.random.default_rng(M + K)
    a, w, sa, sw = operands(rng, M, K, N, q)
    pitch = (K + 15) // 16 * 16
    ap = torch.zeros(M, pitch, dtype=torch.uint8, device="cuda").view(a.dtype)
    ap[:, :K] = a
    sad, one = cu(sa), cu(sa[:1])
    x = torch.randn(64, 1024, device="cuda")
    g, nq, ns = torch.ones(1024, device="cuda"), torch.zeros(64, 1024, dtype=torch.int8, device="cuda"), empty(64)
    with cuda.WeightQ8(w, cu(sw)) as W:
        want, few = empty((M, N)), empty((1, N))
        cuda.wmatmul_q8(ap, sad, W, want)
        check(f64(want), *want_and_tol(a, w, sa, sw, None, None, None, 1.0, "f32", q))
        cuda.wmatmul_q8(ap[:1], one, W, few)
        cuda.residual_rms_norm_q8(x, None, None, 0.0, g, 1e-5, None, nq, ns)
        torch.cuda.synchronize()
        first, nq0 = few.clone(), nq.clone()
        c = [empty((M, N)) for _ in range(3)]
        for i in range(60):
            cuda.wmatmul_q8(ap, sad, W, c[i % 3])
            cuda.wmatmul_q8(ap[:1], one, W, few)
            cuda.residual_rms_norm_q8(x, None, None, 0.0, g, 1e-5, None, nq, ns)
        torch.cuda.synchronize()
        assert all(torch.equal(t, want) for t in c) and torch.equal(few, first) and torch.equal(nq, nq0)
