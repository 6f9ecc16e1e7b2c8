"""What the 8-bit integer operators are measured on: cases, inputs, plain forms and exact values.

The operators quantise symmetrically, one scale for each row ("token") of an
activation and one for each output channel of a weight:

* ``quantize_int8``   q = rn(x * 127 / amax), scale = amax / 127, amax = max_k |x|
* ``rmsnorm_int8``    the same of rmsnorm(x + residual) * gamma, and the sum
* ``matmul_int8``     gelu(scale_m * scale_n * sum_k a_mk b_nk + bias_n) + residual_mn
* ``fused_rmsnorm_matmul_int8``  rmsnorm_int8, then matmul_int8
* ``fused_mlp_int8``  rmsnorm_int8, matmul_int8 with GELU, quantize_int8, matmul_int8 with the residual

Weights are int8 [out, in] with the row stride rounded up to 16 bytes, as
``quantize_int8`` lays them out. Quantised outputs are compared as the bf16
values they stand for.
"""

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-5
MAX_ROWS, MAX_K, MAX_OUT = 8192, 16384, 28672


def _ops():
    try:
        from tfb200 import ops
    except ImportError:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tt-flow_b200"))
        from tfb200 import ops

    return ops


def listed():
    return [
        # The hidden block of one decode step (32 sequences) before its down projection.
        {"name": "quantize_32x28672", "op": "quantize", "M": 32, "K": 28672},
        # The hidden block of a full prefill.
        {"name": "quantize_8192x16384", "op": "quantize", "M": 8192, "K": 16384},
        # One sequence's token in front of a projection: latency only.
        {"name": "rmsnorm_1x4096", "op": "rmsnorm", "M": 1, "K": 4096, "residual": False},
        # Every layer of a prefill: the block's output joins the residual stream and is normalised for the next.
        {"name": "rmsnorm_add_8192x4096", "op": "rmsnorm", "M": 8192, "K": 4096, "residual": True},
        # A decode projection, weights read once.
        {"name": "matmul_32x8192x28672", "op": "matmul", "M": 32, "K": 8192, "N": 28672, "bias": False,
         "gelu": "none", "residual": False, "f32": False},
        # Odd sizes everywhere, fp32 logits of a small classifier head.
        {"name": "matmul_333x1000x517_f32", "op": "matmul", "M": 333, "K": 1000, "N": 517, "bias": True,
         "gelu": "none", "residual": False, "f32": True},
        # An output projection with bias and residual over a prefill's tokens.
        {"name": "matmul_add_8192x4096x4096", "op": "matmul", "M": 8192, "K": 4096, "N": 4096, "bias": True,
         "gelu": "none", "residual": True, "f32": False},
        # The QKV projection of 16 decoding sequences.
        {"name": "norm_matmul_16x4096x6144", "op": "norm_matmul", "M": 16, "K": 4096, "N": 6144},
        # The QKV projection of a prefill.
        {"name": "norm_matmul_8192x4096x6144", "op": "norm_matmul", "M": 8192, "K": 4096, "N": 6144},
        # A single token through an MLP block, exact GELU.
        {"name": "mlp_1x4096x16384_erf", "op": "mlp", "M": 1, "K": 4096, "H": 16384, "N": 4096, "gelu": "erf"},
        # A decode step of 32 sequences through a large MLP block.
        {"name": "mlp_32x8192x28672", "op": "mlp", "M": 32, "K": 8192, "H": 28672, "N": 8192, "gelu": "tanh"},
        # The MLP block of a prefill.
        {"name": "mlp_8192x4096x16384", "op": "mlp", "M": 8192, "K": 4096, "H": 16384, "N": 4096, "gelu": "tanh"},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; about half are multiples of 64, the rest as they fall."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n = (n + 32) // 64 * 64
    return min(max(n, lo), hi)


def draw(rng):
    op = rng.choice(["quantize", "rmsnorm", "matmul", "norm_matmul", "mlp"])
    m = _size(rng, 1, MAX_ROWS)
    if op == "quantize":
        return {"op": op, "M": m, "K": _size(rng, 64, MAX_K)}
    if op == "rmsnorm":
        return {"op": op, "M": m, "K": _size(rng, 64, 8192), "residual": rng.random() < 0.5}
    if op == "matmul":
        return {"op": op, "M": m, "K": _size(rng, 64, MAX_K), "N": _size(rng, 64, 8192),
                "bias": rng.random() < 0.5, "gelu": rng.choice(["none", "none", "erf", "tanh"]),
                "residual": rng.random() < 0.5, "f32": rng.random() < 0.25}
    if op == "norm_matmul":
        return {"op": op, "M": m, "K": _size(rng, 64, 8192), "N": _size(rng, 64, 8192)}
    k = _size(rng, 64, 4096)
    return {"op": op, "M": m, "K": k, "H": _size(rng, 64, 16384), "N": k, "gelu": rng.choice(["erf", "tanh"])}


# ------------------------------------------------------------------- inputs


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std)


def _activations(g, m, k):
    """Tokens: N(0, 1), with one channel in 256 six times as large, as residual streams have them."""
    x = _normal(g, m, k)
    x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 256)]] *= 6.0
    return x.bfloat16()


def _gamma(g, k):
    return (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()


def _rows_int8(w):
    """(q, scale) of the rows of w, with the row stride rounded up to 16 bytes."""
    scale = w.abs().amax(1) / 127.0
    q = torch.zeros(w.shape[0], (w.shape[1] + 15) // 16 * 16, dtype=torch.int8, device=w.device)[:, : w.shape[1]]
    q.copy_(torch.round(w / scale[:, None]))
    return q, scale


def _weight(g, n, k):
    return _rows_int8(_normal(g, n, k, std=1.0 / math.sqrt(k)))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c, op, m, k = dict(case), case["op"], case["M"], case["K"]
    s = {"case": c}
    if op == "matmul":
        s["a"], s["a_scale"] = _rows_int8(_activations(g, m, k).float())
    else:
        s["x"] = _activations(g, m, k)
    if op in ("rmsnorm", "norm_matmul", "mlp"):
        s["gamma"] = _gamma(g, k)
    if op in ("matmul", "norm_matmul"):
        s["w"], s["w_scale"] = _weight(g, c["N"], k)
    s["bias"] = s["residual"] = None
    if op == "matmul" and c["bias"]:
        s["bias"] = _normal(g, c["N"], std=0.02).bfloat16()
    if c.get("residual"):
        s["residual"] = _normal(g, m, c.get("N", k)).bfloat16()
    if op == "mlp":
        s["w1"], s["w1_scale"] = _weight(g, c["H"], k)
        s["b1"] = _normal(g, c["H"], std=0.02).bfloat16()
        s["w2"], s["w2_scale"] = _weight(g, c["N"], c["H"])
        s["residual"] = s["x"]  # the block's own input
    return s


# -------------------------------------------------------------- plain forms


def _stands_for(q, scale):
    y = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    return torch.mul(q, scale[:, None], out=y)


def _quantize(t):
    """fp32 rows -> (rounded values, their largest magnitude)."""
    amax = t.abs().amax(1)
    r = torch.where(amax > 0, 127.0 / amax, torch.zeros_like(amax))
    return torch.round(t * r[:, None]), amax


def _gelu(v, kind):
    if kind == "erf":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if kind == "tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _norm(x, gamma, residual=None):
    s = x.float() if residual is None else x.float() + residual.float()
    inv = 1.0 / torch.sqrt((s * s).mean(1) + EPS)
    q, amax = _quantize(s * gamma.float())
    return s, q, amax * (inv / 127.0)


def _product(q, scale, w, w_scale, bias=None, gelu="none", residual=None):
    v = (q.float() @ w.float().t()) * scale[:, None] * w_scale
    if bias is not None:
        v = v + bias.float()
    v = _gelu(v, gelu)
    return v if residual is None else v + residual.float()


def _run_plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "quantize":
        q, amax = _quantize(s["x"].float())
        scale = amax / 127.0
        return {"y": _stands_for(q, scale), "scale": scale}
    if op == "rmsnorm":
        t, q, scale = _norm(s["x"], s["gamma"], s["residual"])
        out = {"y": _stands_for(q, scale), "scale": scale}
        if c["residual"]:
            out["sum"] = t.bfloat16()
        return out
    if op == "matmul":
        v = _product(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], c["gelu"], s["residual"])
        return v if c["f32"] else v.bfloat16()
    _, q, scale = _norm(s["x"], s["gamma"])
    if op == "norm_matmul":
        return _product(q, scale, s["w"], s["w_scale"]).bfloat16()
    h, amax = _quantize(_product(q, scale, s["w1"], s["w1_scale"], s["b1"], c["gelu"]))
    return _product(h, amax / 127.0, s["w2"], s["w2_scale"], residual=s["residual"]).bfloat16()


def _run_own(s):
    ops, c, op = _ops(), s["case"], s["case"]["op"]
    if op == "quantize":
        q, scale = ops.quantize_int8(s["x"])
        return {"y": _stands_for(q, scale), "scale": scale}
    if op == "rmsnorm":
        if c["residual"]:
            q, scale, t = ops.rmsnorm_int8(s["x"], s["gamma"], EPS, residual=s["residual"])
            return {"y": _stands_for(q, scale), "scale": scale, "sum": t}
        q, scale = ops.rmsnorm_int8(s["x"], s["gamma"], EPS)
        return {"y": _stands_for(q, scale), "scale": scale}
    if op == "matmul":
        return ops.matmul_int8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], gelu=c["gelu"],
                               residual=s["residual"], out_dtype=torch.float32 if c["f32"] else torch.bfloat16)
    if op == "norm_matmul":
        return ops.fused_rmsnorm_matmul_int8(s["x"], s["gamma"], s["w"], s["w_scale"], EPS)
    return ops.fused_mlp_int8(s["x"], s["gamma"], s["w1"], s["w1_scale"], s["b1"], s["w2"], s["w2_scale"],
                              s["residual"], EPS, gelu=c["gelu"])


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# --------------------------------------------------------------------- work


def work(case):
    c, op, m, k = case, case["op"], case["M"], case["K"]
    if op == "quantize":
        return {"bytes": m * k * 3 + m * 4, "flops": 3 * m * k}
    if op == "rmsnorm":
        return {"bytes": m * k * (7 if c["residual"] else 3) + 2 * k + m * 4, "flops": 6 * m * k}
    if op == "matmul":
        n = c["N"]
        out = m * n * ((4 if c["f32"] else 2) + (2 if c["residual"] else 0)) + (2 * n if c["bias"] else 0)
        return {"bytes": m * k + 4 * m + n * k + 4 * n + out, "flops": 2 * m * n * k}
    if op == "norm_matmul":
        n = c["N"]
        return {"bytes": 2 * m * k + 2 * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    h, n = c["H"], c["N"]
    # The residual is the block's input: read once.
    return {"bytes": 2 * m * k + 2 * k + h * k + 6 * h + n * h + 4 * n + 2 * m * n, "flops": 2 * m * h * (k + n)}


# -------------------------------------------------------------------- exact


def exact(case, seed):
    """The definitions in 64 bits; sums of integer products are exact."""
    s, op, f64 = prepare(case, seed), case["op"], torch.float64
    if op == "matmul":
        q, scale = s["a"].to(f64), s["a_scale"].to(f64)
    else:
        total = s["x"].to(f64)
        if op == "rmsnorm" and case["residual"]:
            total = total + s["residual"].to(f64)
        y = total
        if op != "quantize":
            y = total / (total.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["gamma"].to(f64)
        scale = y.abs().max(-1).values / 127.0
        q = (y / scale.clamp_min(1e-300).unsqueeze(-1)).round()
    if op in ("quantize", "rmsnorm"):
        out = {"y": q * scale.unsqueeze(-1), "scale": scale}
        if op == "rmsnorm" and case["residual"]:
            out["sum"] = total
        return out

    def affine(q, scale, w, w_scale, bias):
        v = torch.einsum("mk,nk->mn", q, w.to(f64)) * torch.outer(scale, w_scale.to(f64))
        return v if bias is None else v + bias.to(f64)

    def activate(v, kind):
        if kind == "erf":
            return v / 2 * torch.special.erfc(-v / math.sqrt(2.0))
        if kind == "tanh":
            return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * v * (1.0 + 0.044715 * v.pow(2)))
        return v

    if op == "mlp":
        h = activate(affine(q, scale, s["w1"], s["w1_scale"], s["b1"]), case["gelu"])
        scale = h.abs().max(-1).values / 127.0
        q = (h / scale.clamp_min(1e-300).unsqueeze(-1)).round()
        return affine(q, scale, s["w2"], s["w2_scale"], None) + s["residual"].to(f64)
    v = affine(q, scale, s["w"], s["w_scale"], s["bias"])
    v = activate(v, case.get("gelu", "none"))
    return v if s["residual"] is None else v + s["residual"].to(f64)
