"""The 8-bit step from a hidden state to the next token, operator by operator:
what is timed and compared, in a plain form (elementary torch operations) and
through the library's entry points.

  norm     x' = x + alpha (y + bias); n = x' gamma / sqrt(mean(x'^2) + eps);
           n in 8 bits (int8 or e4m3) with one scale per row
  product  C = R + r act(s_a[m] s_w[n] sum_k A[m,k] W[k,n] + bias[n]) of 8-bit
           operands
  sample   one token per row of logits: temperature, top-k, top-p, min-p, then
           the inverse of the cumulative distribution at a given number u
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet-unified-en-0.6b-c_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pkcuda
    return pkcuda


# ── cases ────────────────────────────────────────────────────────────────────


def listed():
    norm = dict(op="norm", bias=True, alpha=1.0)
    prod = dict(op="product", bias=True, residual=False, column_scales=False)
    return [
        # one frame of a stream, or one token: latency
        dict(norm, name="norm_1x1024_f32_int8", rows=1, width=1024, dtype="f32", q="int8"),
        # one 30 s utterance (375 encoder frames), the half-step residual of a feed-forward module
        dict(norm, name="norm_375x1024_f32_e4m3", rows=375, width=1024, dtype="f32", q="e4m3", alpha=0.5),
        # a batch of 32 utterances
        dict(norm, name="norm_12000x1024_f32_int8", rows=12000, width=1024, dtype="f32", q="int8", alpha=0.5),
        # a wide model's 16-bit stream, an odd number of rows, no bias
        dict(norm, name="norm_2049x8192_bf16_e4m3", rows=2049, width=8192, dtype="bf16", q="e4m3", bias=False),
        # one token through a feed-forward projection: the weight's bytes count
        dict(prod, name="product_1x1024x4096_int8", m=1, k=1024, n=4096, q="int8", act="swish", dtype="bf16"),
        # the joint's output projection for 32 utterances: 1025 logits, rows of odd length
        dict(prod, name="product_32x640x1025_int8", m=32, k=640, n=1025, q="int8", act="none", dtype="f32"),
        # the first feed-forward projection of 32 utterances
        dict(prod, name="product_12000x1024x4096_int8", m=12000, k=1024, n=4096, q="int8", act="swish", dtype="bf16", column_scales=True),
        # the second one, with the half-step residual, in fp32 as the encoder's stream is
        dict(prod, name="product_12000x4096x1024_int8", m=12000, k=4096, n=1024, q="int8", act="none", dtype="f32", residual=True),
        # a wide model's projection, in floating 8 bits
        dict(prod, name="product_2049x8192x8192_e4m3", m=2049, k=8192, n=8192, q="e4m3", act="gelu", dtype="bf16", column_scales=True),
        # one token of a large vocabulary, top-p
        dict(op="sample", name="sample_1x131072_bf16_top_p", rows=1, vocab=131072, dtype="bf16", mode="top_p", masked=0.0),
        # every frame's draw from the joint's 1025 logits, top-k
        dict(op="sample", name="sample_12000x1025_f32_top_k", rows=12000, vocab=1025, dtype="f32", mode="top_k", masked=0.0),
        # a serving batch, each row with its own settings, some tokens forbidden
        dict(op="sample", name="sample_256x32000_f32_mixed", rows=256, vocab=32000, dtype="f32", mode="mixed", masked=0.05),
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("norm", "product", "sample"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "norm":
        width = size(64, 8192)
        return dict(op=op, rows=size(1, min(12000, 16_000_000 // width)), width=width, dtype=dtype, q=rng.choice(("int8", "e4m3")),
                    bias=rng.random() < 0.5, alpha=rng.choice((0.5, 1.0)))
    if op == "product":
        k, n = size(64, 8192), size(32, 8192)
        return dict(op=op, m=size(1, max(1, min(12000, 48_000_000 // n, 50_000_000_000 // (k * n)))), k=k, n=n, q=rng.choice(("int8", "e4m3")),
                    act=rng.choice(("none", "relu", "swish", "gelu", "tanh")), dtype=dtype, bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5, column_scales=rng.random() < 0.5)
    vocab = size(32, 131072)
    return dict(op=op, rows=size(1, min(12000, 8_000_000 // vocab)), vocab=vocab, dtype=dtype,
                mode=rng.choice(("plain", "top_k", "top_p", "min_p", "mixed")), masked=rng.choice((0.0, 0.05, 0.5)))


# ── inputs ───────────────────────────────────────────────────────────────────


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        t = DTYPES[case["dtype"]]
        s["x"] = (2.0 * normal(rows, width)).to(t)
        s["y"] = normal(rows, width).to(t)
        s["b"] = 0.1 * normal(width) if case["bias"] else None
        s["gamma"] = 1.0 + 0.2 * normal(width)
        s["pitch"] = -(-width // 16) * 16
        s["x_out"] = torch.empty_like(s["x"])
        s["q_out"] = torch.zeros(rows, s["pitch"], dtype=_q_type(case["q"]), device="cuda")
        s["scales"] = torch.empty(rows, device="cuda")
        s["values"] = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda") if case["q"] == "int8" else None
    elif case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        t = DTYPES[case["dtype"]]
        pitch = -(-k // 16) * 16
        s["a"] = torch.zeros(m, pitch, dtype=_q_type(case["q"]), device="cuda")
        s["a"][:, :k] = _in_8_bits(normal(m, k), case["q"])
        s["w"] = _in_8_bits(normal(k, n), case["q"])
        top = 127.0 if case["q"] == "int8" else 448.0
        s["a_scales"] = (3.0 + uniform(m)) / top
        s["w_scales"] = (3.0 + uniform(n if case["column_scales"] else 1)) / (top * math.sqrt(k))
        s["b"] = 0.5 * normal(n) if case["bias"] else None
        s["r"] = normal(m, n).to(t) if case["residual"] else None
        s["out"] = torch.empty(m, n, dtype=t, device="cuda")
        if own:  # a program keeps its weights laid out for the products
            s["weight"] = _lib().WeightQ8(s["w"], s["w_scales"])
    else:
        rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
        x = 2.5 * normal(rows, vocab) + 6.0 * (uniform(rows, vocab) < 8.0 / vocab)
        if case["masked"]:
            x = x.masked_fill(uniform(rows, vocab) < case["masked"], -math.inf)
            x[:, seed % vocab] = 1.0  # a row keeps something
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["temperature"] = 0.6 + 0.6 * uniform(rows)
        k = (1 + 99 * uniform(rows)).to(torch.int32)
        p = 0.5 + 0.49 * uniform(rows)
        q = 0.01 + 0.2 * uniform(rows)
        pick = torch.arange(rows, device="cuda") % 4  # mixed: a row in four has no filter of a kind, and one is greedy
        if mode == "mixed":
            k[pick == 1] = 0
            p[pick == 2] = 1.0
            q[pick != 3] = 0.0
            s["temperature"][torch.arange(rows, device="cuda") % 16 == 5] = 0.0
        s["top_k"] = k if mode in ("top_k", "mixed") else None
        s["top_p"] = p if mode in ("top_p", "mixed") else None
        s["min_p"] = q if mode in ("min_p", "mixed") else None
        s["u"] = uniform(rows)
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(rows, device="cuda")
    return s


def _q_type(q):
    return torch.int8 if q == "int8" else torch.float8_e4m3fn


def _in_8_bits(x, q):
    """Values of N(0, 1) at a scale of four standard deviations."""
    if q == "int8":
        return (x * (127.0 / 4.0)).round().clamp(-127, 127).to(torch.int8)
    return (x * (448.0 / 4.0)).clamp(-448, 448).to(torch.float8_e4m3fn)


# ── one pass ─────────────────────────────────────────────────────────────────


def run(s):
    return {"norm": _norm, "product": _product, "sample": _sample}[s["op"]](s)


def _stands_for(s, q, scales):
    """The 8-bit values: e4m3 as they are (a floating type, its scales beside
    them), int8 as what they stand for, in 16 bits."""
    if s["q"] == "e4m3":
        return q
    return torch.mul(q, scales[:, None], out=s["values"])


def _norm(s):
    if own:
        _lib().residual_rms_norm_q8(s["x"], s["y"], s["b"], s["alpha"], s["gamma"], EPS, s["x_out"], s["q_out"], s["scales"])
        return [s["x_out"], _stands_for(s, s["q_out"][:, :s["width"]], s["scales"]), s["scales"]]
    y = s["y"].float()
    if s["b"] is not None:
        y = y + s["b"]
    x_out = (s["x"].float() + s["alpha"] * y).to(s["x"].dtype)
    x = x_out.float()
    n = x * s["gamma"] / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS)
    top = 127.0 if s["q"] == "int8" else 448.0
    scales = n.abs().amax(dim=1) / top
    v = n / scales[:, None]
    v = v.round().to(torch.int8) if s["q"] == "int8" else v.clamp(-448, 448).to(torch.float8_e4m3fn)
    return [x_out, _stands_for(s, v, scales), scales]


def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "swish":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "tanh":
        return torch.tanh(v)
    return v


def _product(s):
    if own:
        _lib().wmatmul_q8(s["a"], s["a_scales"], s["weight"], s["out"], bias=s["b"], act=s["act"], residual=s["r"], rscale=0.5 if s["residual"] else 1.0)
        return s["out"]
    v = (s["a"][:, :s["k"]].float() @ s["w"].float()) * s["a_scales"][:, None] * s["w_scales"][None, :]
    if s["b"] is not None:
        v = v + s["b"]
    v = _act(v, s["act"])
    if s["r"] is not None:
        v = s["r"].float() + 0.5 * v
    return v.to(s["out"].dtype)


def _sample(s):
    if own:
        _lib().sample_rows(s["logits"], s["u"], s["tokens"], s["logprobs"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return [s["tokens"], s["logprobs"]]
    # in 64 bits: a token is a border of the cumulative sum next to u
    x = s["logits"].double()
    rows, vocab = x.shape
    top = x.amax(dim=1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = t[:, 0] <= 0
    w = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    w_sorted, order = torch.sort(w, dim=1, descending=True, stable=True)
    rank = torch.arange(vocab, device=x.device)[None, :]
    keep = torch.ones_like(w_sorted, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (rank < k) | (k <= 0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        c = torch.cumsum(w_sorted * keep, dim=1)
        before = torch.cat([torch.zeros_like(c[:, :1]), c[:, :-1]], dim=1)
        keep &= (before < p * c[:, -1:]) | (p >= 1) | (rank == 0)
    if s["min_p"] is not None:
        keep &= w_sorted >= s["min_p"].double()[:, None].clamp(0, 1)
    kept = torch.zeros_like(w).scatter_(1, order, w_sorted * keep)
    c = torch.cumsum(kept, dim=1)
    total = c[:, -1]
    token = (c <= (s["u"].double() * total)[:, None]).sum(dim=1).clamp_max(vocab - 1)
    first = (x == top).to(torch.int8).argmax(dim=1)
    token = torch.where(greedy, first, token)
    logp = torch.log(kept.gather(1, token[:, None])[:, 0] / total)
    return [token.to(torch.int32), torch.where(greedy, torch.zeros_like(logp), logp).float()]


# ── work and values in 64 bits ───────────────────────────────────────────────


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["width"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * (3 * size + 1) + 4 * case["rows"] + 4 * case["width"] * (1 + case["bias"]), "flops": 8 * n}
    if case["op"] == "product":
        m, k, n, size = case["m"], case["k"], case["n"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": m * k + k * n + m * n * size * (1 + case["residual"]) + 4 * (m + n * (case["column_scales"] + case["bias"])), "flops": 2 * m * k * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 28 * case["rows"], "flops": 4 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        t = DTYPES[case["dtype"]]
        add = s["y"].double() if s["b"] is None else s["y"].double() + s["b"].double()
        x_out = s["x"].double() + case["alpha"] * add
        x = x_out.to(t).double()  # the norm is of what is stored
        r = (x.pow(2).sum(dim=1) / case["width"] + EPS).rsqrt()
        n = x * r[:, None] * s["gamma"].double()
        scales = n.abs().max(dim=1).values / (127 if case["q"] == "int8" else 448)
        v = n / scales[:, None]
        v = torch.round(v) if case["q"] == "int8" else v.float().to(torch.float8_e4m3fn).double()
        return [x_out, v * scales[:, None] if case["q"] == "int8" else v, scales]
    if case["op"] == "product":
        v = torch.matmul(s["a"].double()[:, :case["k"]], s["w"].double())
        v = v * torch.outer(s["a_scales"].double(), s["w_scales"].double().expand(case["n"]))
        if case["bias"]:
            v += s["b"].double()
        if case["act"] == "relu":
            v = torch.where(v > 0, v, 0.0)
        elif case["act"] == "swish":
            v = v * torch.sigmoid(v)
        elif case["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        elif case["act"] == "tanh":
            v = 1 - 2 / (torch.exp(2 * v) + 1)
        return v if not case["residual"] else s["r"].double() + v / 2
    host = {k: v.cpu().double().numpy() if torch.is_tensor(v) else v for k, v in s.items()}
    tokens, logprobs = [], []
    for i, x in enumerate(host["logits"]):
        t = host["temperature"][i]
        if t <= 0:
            tokens.append(int(np.argmax(x)))
            logprobs.append(0.0)
            continue
        p = np.exp((x - x.max()) / t)
        by = np.argsort(-x, kind="stable")
        if host["top_k"] is not None and host["top_k"][i] > 0:
            by = by[: int(host["top_k"][i])]
        if host["top_p"] is not None and host["top_p"][i] < 1:
            c = np.cumsum(p[by])
            by = by[: 1 + int(np.searchsorted(c, host["top_p"][i] * c[-1], side="left"))]
        if host["min_p"] is not None:
            by = by[p[by] >= min(max(host["min_p"][i], 0.0), 1.0)]
        by = np.sort(by)
        c = np.cumsum(p[by])
        at = min(int(np.searchsorted(c, host["u"][i] * c[-1], side="right")), len(by) - 1)
        tokens.append(int(by[at]))
        logprobs.append(float(np.log(p[by[at]] / c[-1])))
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)]
