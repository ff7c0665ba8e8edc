"""GPU: the 8-bit operators in a row, as a decoder's last block and head run
them: residual + norm (8 bits) -> product with Swish -> ... -> residual + norm ->
product to logits -> one drawn token per row; on one stream, and captured into
one graph that is replayed on new inputs.

Each step is checked on the GPU's own inputs to it: norms and products within
their tests' tolerances, tokens equal to the definition's on the GPU's logits."""
import numpy as np
import pytest

from gpuhelp import empty
from q8help import cu, f64, rms_q8
from test_sample_rows_gpu import plain
from test_wmatmul_q8_gpu import check as check_close, want_and_tol

pytestmark = pytest.mark.gpu

D, FF, V, EPS = 1024, 4096, 1025, 1e-5


class Chain:
    def __init__(self, cuda, rows, q, seed):
        import torch
        r = np.random.default_rng(seed)
        n = lambda *s: cu(r.standard_normal(s).astype(np.float32))
        self.cuda, self.rows, self.q = cuda, rows, q
        t = torch.int8 if q == "i8" else torch.float8_e4m3fn
        lim = 127 if q == "i8" else 448

        def weight(K, N):
            w = r.standard_normal((K, N)) * (lim / 4)
            w = cu(np.clip(np.rint(w) if q == "i8" else w, -lim, lim).astype(np.float32)).to(t)
            return w, np.full(N, 4 / lim / np.sqrt(K), np.float32)

        self.x, self.y = n(rows, D), n(rows, D)
        self.gammas = [cu((1 + 0.1 * r.standard_normal(D)).astype(np.float32)) for _ in range(2)]
        self.raw = [weight(D, FF), weight(FF, D), weight(D, V)]
        self.w = [cuda.WeightQ8(w, cu(s)) for w, s in self.raw]
        self.b = [n(FF), n(D), n(V)]
        e8 = lambda cols: empty((rows, cols), torch.uint8).view(t)
        self.x1, self.x2 = empty((rows, D)), empty((rows, D))
        self.q1, self.s1, self.q2, self.s2 = e8(D), empty(rows), e8(D), empty(rows)
        self.h, self.hq, self.hs = empty((rows, FF)), e8(FF), empty(rows)
        self.ones = cu(np.ones(FF, np.float32))
        self.logits = empty((rows, V))
        self.u = cu(r.random(rows).astype(np.float32))
        self.p = cu(np.full(rows, 0.9, np.float32))
        self.k = cu(np.full(rows, 50, np.int32))
        self.tok, self.lp = empty(rows, torch.int32), empty(rows)

    def run(self):
        c = self.cuda
        c.residual_rms_norm_q8(self.x, self.y, None, 0.5, self.gammas[0], EPS, self.x1, self.q1, self.s1)
        c.wmatmul_q8(self.q1, self.s1, self.w[0], self.h, bias=self.b[0], act="swish")
        c.residual_rms_norm_q8(self.h, None, None, 0.0, self.ones, EPS, None, self.hq, self.hs)
        c.wmatmul_q8(self.hq, self.hs, self.w[1], self.x2, bias=self.b[1], residual=self.x1, rscale=0.5)
        c.residual_rms_norm_q8(self.x2, None, None, 0.0, self.gammas[1], EPS, None, self.q2, self.s2)
        c.wmatmul_q8(self.q2, self.s2, self.w[2], self.logits, bias=self.b[2])
        c.sample_rows(self.logits, self.u, self.tok, self.lp, top_k=self.k, top_p=self.p)

    def check(self):
        Q = 127.0 if self.q == "i8" else 448.0
        for x, g, q, s in ((self.x1, self.gammas[0], self.q1, self.s1), (self.h, self.ones, self.hq, self.hs),
                           (self.x2, self.gammas[1], self.q2, self.s2)):
            ws, v = rms_q8(f64(x), f64(g), EPS, Q)
            assert np.allclose(f64(s), ws, rtol=2e-5, atol=0)
            step = 0.5001 if self.q == "i8" else np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10) * 1.00001
            assert (np.abs(f64(q) - v) <= step).all()
        for i, (a, s, act, r, rs, out) in enumerate(((self.q1, self.s1, "swish", None, 1.0, self.h),
                                                     (self.hq, self.hs, None, self.x1, 0.5, self.x2),
                                                     (self.q2, self.s2, None, None, 1.0, self.logits))):
            w, sw = self.raw[i]
            want, tol = want_and_tol(a, w, f64(s).astype(np.float32), sw, f64(self.b[i]).astype(np.float32), act, r, rs,
                                     "f32", self.q)
            check_close(f64(out), want, tol, f"product {i}")
        x, u, tok = f64(self.logits), f64(self.u), f64(self.tok)
        for i in range(self.rows):
            assert plain(x[i], u[i], 1.0, 50, float(np.float32(0.9)), 0.0)[0] == tok[i]


@pytest.mark.parametrize("q", ["i8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 5, 64, 375])
def test_chain(cuda, rows, q):
    import torch
    c = Chain(cuda, rows, q, rows)
    c.run()
    c.check()
    tokens = c.tok.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    c.tok.fill_(-9)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.tok, tokens)
    c.x.mul_(-1.0)
    c.u.copy_(1 - c.u)
    g.replay()
    c.check()
    for w in c.w:
        w.close()


def test_two_graphs_and_an_eager_call(cuda):
    """Two captured chains replayed on two streams while a third runs eagerly."""
    import torch
    chains = [Chain(cuda, 32, "i8", s) for s in (1, 2, 3)]
    want = []
    for c in chains:
        c.run()
        torch.cuda.synchronize()
        want.append((c.tok.clone(), c.logits.clone()))
    graphs = []
    for c in chains[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        chains[2].run()
    torch.cuda.synchronize()
    for c, (t, l) in zip(chains, want):
        assert torch.equal(c.tok, t) and torch.equal(c.logits, l)
        for w in c.w:
            w.close()
