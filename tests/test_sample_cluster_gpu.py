"""GPU: pkcu_sample_rows where a row is a cluster's and top-k takes nothing away:
top_k is the row's length, or at least the number of its entries that are left by
the mask, and top-p follows. The cluster then fills its bins a second time, and
every CTA has to be done with reading them first.

Tokens have to be equal to the definition's, and to themselves over many calls."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu
from test_sample_rows_gpu import check

pytestmark = pytest.mark.gpu


def rows_with(rng, rows, V, live):
    """Rows of V logits with `live` entries left, spread over the whole row (None: all)."""
    x = (3 * rng.standard_normal((rows, V))).astype(np.float32)
    if live is not None:
        keep = np.zeros((rows, V), bool)
        for r in range(rows):
            keep[r, np.unique(np.linspace(0, V - 1, live).astype(int) if r % 2 else rng.integers(0, V, live))] = True
        x[~keep] = -np.inf
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("live", [None, 1, 40, 3000])
@pytest.mark.parametrize("rows,V", [(1, 20000), (4, 40000), (2, 131072), (40, 65536), (1, 262144)])
def test_top_k_of_all_then_top_p(cuda, rows, V, live, dtype):
    rng = np.random.default_rng(V + rows + (live or 0))
    x = cu(rows_with(rng, rows, V, live), dtype)
    u = rng.random(rows).astype(np.float32)
    for k in (V, V - 1, live or V, (live or V) + 1, 2 ** 31 - 1):
        for p in (0.9, 0.3):
            check(cuda, x, u, k=np.full(rows, k), p=np.full(rows, p), what=f"k {k} p {p}")


def test_repeats(cuda):
    """Different ways through the filters in neighbouring rows, many times over."""
    import torch
    rng = np.random.default_rng(0)
    rows, V = 12, 100000
    x = rows_with(rng, rows, V, None)
    x[::3, 5000:] = -np.inf            # all that is left in the first CTA
    x[1::3, :-70] = -np.inf            # ... in the last
    x = cu(x)
    u = rng.random(rows).astype(np.float32)
    k = np.resize(np.array([V, 70, 5000, 50]), rows)
    want, _ = check(cuda, x, u, k=k, p=np.full(rows, 0.9))
    kd, pd, ud = cu(k.astype(np.int32)), cu(np.full(rows, 0.9, np.float32)), cu(u)
    outs = [empty(rows, torch.int32) for _ in range(200)]
    for t in outs:
        cuda.sample_rows(x, ud, t, top_k=kd, top_p=pd)
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in outs)
