"""The operators of a transformer block's training step, as cases to be timed.

A case is one call of one operator at one shape:

* ``ln``       ``layer_norm`` over rows, with weight and bias
* ``ln_bwd``   its gradients: the input's, the weight's and the bias's
* ``mm``       ``matmul_epilogue``: a product with bias, activation and residual
* ``mm_bwd``   its gradients: both operands' and the bias's
* ``ns``       ``newton_schulz``: an update matrix orthogonalised, as the Muon optimiser does

Where ``own`` is false the operators are computed from elementary torch
operations in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

KINDS = ("ln", "ln_bwd", "mm", "mm_bwd", "ns")
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
EPS = 1e-5
NS_STEPS = 5
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7

MAX_LN = 16384 * 8192  # elements of the largest normalised tensor
MAX_MM = 8192**3  # multiply-adds of the largest product
MAX_MM_BWD = 4096**3
MAX_OPERAND = 28672 * 8192  # elements of the largest weight
MAX_NS = 4096**3  # batch * m * m * n of the largest update


def _ln(name: str, kind: str, rows: int, D: int, dtype: str, weight: str) -> dict:
    return {"name": name, "kind": kind, "rows": rows, "D": D, "dtype": dtype, "weight": weight}


def _mm(name: str, kind: str, M: int, N: int, K: int, act: str, bias: str, residual: bool, transposed: bool,
        pre: bool = False) -> dict:
    return {"name": name, "kind": kind, "M": M, "N": N, "K": K, "act": act, "bias": bias, "residual": residual,
            "transposed": transposed, "pre": pre}


def _ns(name: str, batch: int, m: int, n: int, dtype: str) -> dict:
    return {"name": name, "kind": "ns", "batch": batch, "m": m, "n": n, "dtype": dtype}


def listed() -> list[dict]:
    return [
        # The norm of a few decoded rows: latency bound, the smallest call.
        _ln("ln_decode", "ln", 8, 4096, "bfloat16", "bfloat16"),
        # The norm of a long prefill: bound by reading and writing the rows.
        _ln("ln_prefill", "ln", 16384, 8192, "bfloat16", "bfloat16"),
        # Gradients at sizes that are no multiple of anything, all in fp32.
        _ln("ln_bwd_ragged", "ln_bwd", 1000, 1501, "float32", "float32"),
        # Gradients of a large training batch; master weights in fp32.
        _ln("ln_bwd_train", "ln_bwd", 16384, 4096, "bfloat16", "float32"),
        # Decode of 16 rows against a large weight: bound by reading it.
        _mm("mm_decode", "mm", 16, 28672, 8192, "silu", "bfloat16", False, False),
        # A down projection of a ragged number of rows, added to the residual stream; weight [N, K].
        _mm("mm_residual", "mm", 1000, 5000, 4104, "none", "bfloat16", True, True),
        # The first layer of a large MLP in training: the pre-activation is kept for the backward pass.
        _mm("mm_train", "mm", 8192, 8192, 8192, "gelu_tanh", "bfloat16", False, False, True),
        # Gradients at odd sizes (no dimension a multiple of 8).
        _mm("mm_bwd_ragged", "mm_bwd", 1000, 1501, 777, "gelu", "float32", False, True),
        # Gradients of a training batch.
        _mm("mm_bwd_train", "mm_bwd", 4096, 4096, 4096, "gelu_tanh", "bfloat16", False, False),
        # Updates of a few small projections of one shape, as one batch.
        _ns("ns_small", 4, 256, 512, "bfloat16"),
        # A tall update at odd sizes, gradients kept in fp32.
        _ns("ns_tall", 1, 2001, 777, "float32"),
        # The update of a large square projection.
        _ns("ns_large", 1, 4096, 4096, "bfloat16"),
    ]


def _spread(rng, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of ``step`` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng) -> dict:
    kind = rng.choice(KINDS)
    if kind in ("ln", "ln_bwd"):
        while True:
            rows, D = _spread(rng, 1, 65536), _spread(rng, 8, 32768, rng.choice((1, 8, 64)))
            if 4096 <= rows * D <= MAX_LN // (1 if kind == "ln" else 2):
                break
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        return {"kind": kind, "rows": rows, "D": D, "dtype": dtype, "weight": rng.choice((dtype, "float32"))}
    if kind in ("mm", "mm_bwd"):
        while True:
            M = _spread(rng, 1, 8192, rng.choice((1, 8)))
            N, K = (_spread(rng, 64, 28672, rng.choice((1, 8, 8, 64))) for _ in range(2))
            if N * K <= MAX_OPERAND and M * N * K <= (MAX_MM if kind == "mm" else MAX_MM_BWD):
                break
        return {"kind": kind, "M": M, "N": N, "K": K, "act": rng.choice(ACTIVATIONS),
                "bias": rng.choice(("", "bfloat16", "bfloat16", "float32")),
                "residual": kind == "mm" and rng.random() < 0.5, "transposed": rng.random() < 0.5,
                "pre": kind == "mm" and rng.random() < 0.3}
    while True:
        batch = rng.choice((1, 1, 1, 2, 4, 8))
        m, n = (_spread(rng, 32, 8192, rng.choice((1, 8, 64))) for _ in range(2))
        if batch * min(m, n) ** 2 * max(m, n) <= MAX_NS:
            break
    return {"kind": "ns", "batch": batch, "m": m, "n": n, "dtype": rng.choice(("bfloat16", "float32"))}


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=dev) * std

    s = {"case": case}
    kind = case["kind"]
    if kind in ("ln", "ln_bwd"):
        rows, D, dtype, wt = case["rows"], case["D"], DTYPES[case["dtype"]], DTYPES[case["weight"]]
        # A residual stream: rows of their own mean and spread.
        x = normal(rows, D)
        x *= 0.5 + torch.rand((rows, 1), generator=gen, device=dev)
        x += 0.5 + 0.2 * normal(rows, 1)
        s["x"] = x.to(dtype)
        s["weight"] = (1 + 0.1 * normal(D)).to(wt)
        s["bias"] = (0.1 * normal(D)).to(wt)
        if kind == "ln_bwd":
            s["dout"] = normal(rows, D, std=0.1).to(dtype)
            # What the forward call left for its backward pass.
            xd = s["x"].double()
            mean = xd.mean(dim=1)
            var = xd.sub_(mean[:, None]).square_().mean(dim=1)
            s["mean"], s["rstd"] = mean.float(), (var + EPS).rsqrt().float()
    elif kind in ("mm", "mm_bwd"):
        M, N, K = case["M"], case["N"], case["K"]
        bf16 = torch.bfloat16
        s["lhs"] = normal(M, K).to(bf16)
        s["rhs"] = normal(*((N, K) if case["transposed"] else (K, N)), std=1 / math.sqrt(K)).to(bf16)
        s["bias"] = normal(N, std=0.1).to(DTYPES[case["bias"]]) if case["bias"] else None
        if kind == "mm":
            s["residual"] = normal(M, N).to(bf16) if case["residual"] else None
        else:
            s["dout"] = normal(M, N, std=0.1).to(bf16)
            s["pre"] = normal(M, N).to(bf16) if case["act"] != "none" else None
    else:
        batch, m, n = case["batch"], case["m"], case["n"]
        # A gradient: a part of low rank and noise.
        r = max(1, min(m, n) // 16)
        g = torch.matmul(normal(batch, m, r), normal(batch, r, n, std=1 / math.sqrt(r))) + normal(batch, m, n)
        s["grad"] = (1e-3 * g).to(DTYPES[case["dtype"]])
    return s


def _kl():
    path = os.path.join(os.getcwd(), "nki-autotune_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kernel_library

    return kernel_library


def _run_own(s: dict):
    kl, c = _kl(), s["case"]
    if c["kind"] == "ln":
        y, mean, rstd = kl.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, stats=True)
        return {"y": y, "mean": mean, "rstd": rstd}
    if c["kind"] == "ln_bwd":
        dx, dweight, dbias = kl.layer_norm_backward(s["dout"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"])
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    if c["kind"] == "mm":
        pre = torch.empty((c["M"], c["N"]), dtype=torch.bfloat16, device=s["lhs"].device) if c["pre"] else None
        out = kl.matmul_epilogue(s["lhs"], s["rhs"], s["bias"], c["act"], s["residual"],
                                 rhs_transposed=c["transposed"], pre=pre)
        return {"out": out, "pre": pre} if c["pre"] else {"out": out}
    if c["kind"] == "mm_bwd":
        dlhs, drhs, dbias = kl.matmul_epilogue_backward(s["dout"], s["lhs"], s["rhs"], c["act"], s["pre"], s["bias"],
                                                        rhs_transposed=c["transposed"])
        return {"dlhs": dlhs, "drhs": drhs, "dbias": dbias} if c["bias"] else {"dlhs": dlhs, "drhs": drhs}
    return {"out": kl.newton_schulz(s["grad"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS, eps=NS_EPS)}


def _act(act: str, x: torch.Tensor) -> torch.Tensor:
    if act == "relu":
        return torch.clamp_min(x, 0.0)
    if act == "gelu":
        return 0.5 * x * torch.erfc(-x * math.sqrt(0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    return x


def _act_grad(act: str, x: torch.Tensor) -> torch.Tensor:
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "gelu":
        return 0.5 * torch.erfc(-x * math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x * x * x))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * x * x)
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-x))
        return sg * (1.0 + x * (1.0 - sg))
    return torch.ones_like(x)


def run(s: dict):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["kind"] == "ln":
        x = s["x"].float()
        mean = x.mean(dim=1)
        xc = x - mean[:, None]
        rstd = torch.rsqrt((xc * xc).mean(dim=1) + EPS)
        y = xc * rstd[:, None] * s["weight"].float() + s["bias"].float()
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    if c["kind"] == "ln_bwd":
        xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        dy = s["dout"].float()
        g = dy * s["weight"].float()
        dx = s["rstd"][:, None] * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
        wt = s["weight"].dtype
        return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(dim=0).to(wt), "dbias": dy.sum(dim=0).to(wt)}
    if c["kind"] == "mm":
        rhs = s["rhs"].float()
        pre = s["lhs"].float() @ (rhs.t() if c["transposed"] else rhs)
        if s["bias"] is not None:
            pre = pre + s["bias"].float()
        out = _act(c["act"], pre)
        if s["residual"] is not None:
            out = out + s["residual"].float()
        out = out.to(torch.bfloat16)
        return {"out": out, "pre": pre.to(torch.bfloat16)} if c["pre"] else {"out": out}
    if c["kind"] == "mm_bwd":
        dpre = s["dout"].float()
        if s["pre"] is not None:
            dpre = dpre * _act_grad(c["act"], s["pre"].float())
        lhs, rhs = s["lhs"].float(), s["rhs"].float()
        if c["transposed"]:
            dlhs, drhs = dpre @ rhs, dpre.t() @ lhs
        else:
            dlhs, drhs = dpre @ rhs.t(), lhs.t() @ dpre
        grads = {"dlhs": dlhs.to(torch.bfloat16), "drhs": drhs.to(torch.bfloat16)}
        if s["bias"] is not None:
            grads["dbias"] = dpre.sum(dim=0).to(s["bias"].dtype)
        return grads
    a, b, k = NS_COEFFICIENTS
    x = s["grad"].float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (torch.sqrt((x * x).sum(dim=(-2, -1), keepdim=True)) + NS_EPS)
    for _ in range(NS_STEPS):
        A = torch.matmul(x, x.mT.contiguous())
        x = a * x + torch.matmul(b * A + k * torch.matmul(A, A), x.contiguous())
    return {"out": (x.mT if tall else x).to(torch.bfloat16).contiguous()}


def work(case: dict) -> dict:
    kind = case["kind"]
    size = {"": 0, "bfloat16": 2, "float16": 2, "float32": 4}
    if kind in ("ln", "ln_bwd"):
        rows, D, e, w = case["rows"], case["D"], size[case["dtype"]], size[case["weight"]]
        if kind == "ln":
            return {"bytes": 2 * rows * D * e + 2 * D * w + 8 * rows, "flops": 8 * rows * D}
        return {"bytes": 3 * rows * D * e + 8 * rows + 3 * D * w, "flops": 14 * rows * D}
    if kind in ("mm", "mm_bwd"):
        M, N, K, b = case["M"], case["N"], case["K"], size[case["bias"]]
        operands = 2 * (M * K + K * N)
        if kind == "mm":
            return {"bytes": operands + 2 * M * N * (1 + case["residual"] + case["pre"]) + N * b, "flops": 2 * M * N * K}
        return {"bytes": 2 * operands + 2 * M * N * (1 + (case["act"] != "none")) + N * b, "flops": 4 * M * N * K}
    m, n = sorted((case["m"], case["n"]))
    batch = case["batch"]
    # A and A.A are symmetric: half of each, and the diagonal.
    flops = NS_STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
    return {"bytes": batch * m * n * (size[case["dtype"]] + 2), "flops": batch * flops}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f64 = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    kind = case["kind"]
    if kind == "ln":
        mean = f64["x"].mean(dim=1, keepdim=True)
        var = (f64["x"] - mean).pow(2).mean(dim=1, keepdim=True)
        return {"y": (f64["x"] - mean) / torch.sqrt(var + EPS) * f64["weight"] + f64["bias"], "mean": mean[:, 0],
                "rstd": 1 / torch.sqrt(var + EPS)[:, 0]}
    if kind == "ln_bwd":
        D = case["D"]
        centred, rstd = f64["x"] - f64["mean"].unsqueeze(1), f64["rstd"].unsqueeze(1)
        gw = f64["dout"] * f64["weight"]
        along_one = gw.sum(1, keepdim=True) / D
        along_x = (gw * centred).sum(1, keepdim=True) * rstd * rstd / D
        return {"dx": rstd * (gw - along_one - centred * along_x), "dweight": (f64["dout"] * centred * rstd).sum(0),
                "dbias": f64["dout"].sum(0)}
    if kind in ("mm", "mm_bwd"):
        weight = f64["rhs"].t().contiguous() if case["transposed"] else f64["rhs"]
        normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device=weight.device), 1.0)
        root = math.sqrt(2 / math.pi)
        if kind == "mm":
            pre = torch.mm(f64["lhs"], weight)
            if f64["bias"] is not None:
                pre += f64["bias"]
            out = {"none": lambda: pre, "relu": lambda: torch.where(pre > 0, pre, 0.0),
                   "gelu": lambda: pre * normal.cdf(pre),
                   "gelu_tanh": lambda: pre * torch.sigmoid(2 * root * (pre + 0.044715 * pre**3)),
                   "silu": lambda: pre * torch.sigmoid(pre)}[case["act"]]()
            if f64["residual"] is not None:
                out = out + f64["residual"]
            return {"out": out, "pre": pre} if case["pre"] else {"out": out}
        slope, p = 1.0, f64["pre"]
        if case["act"] == "relu":
            slope = torch.where(p > 0, 1.0, 0.0).double()
        elif case["act"] == "gelu":
            slope = normal.cdf(p) + p * torch.exp(normal.log_prob(p))
        elif case["act"] == "gelu_tanh":
            gate = torch.sigmoid(2 * root * (p + 0.044715 * p**3))
            slope = gate + p * gate * (1 - gate) * 2 * root * (1 + 3 * 0.044715 * p**2)
        elif case["act"] == "silu":
            gate = torch.sigmoid(p)
            slope = gate + p * gate * (1 - gate)
        dpre = f64["dout"] * slope
        dweight = torch.mm(f64["lhs"].t().contiguous(), dpre)
        grads = {"dlhs": torch.mm(dpre, weight.t().contiguous()), "drhs": dweight.t().contiguous() if case["transposed"] else dweight}
        if f64["bias"] is not None:
            grads["dbias"] = dpre.sum(0)
        return grads
    out = []
    for g in f64["grad"]:
        flip = g.shape[0] > g.shape[1]
        x = g.t().contiguous() if flip else g
        x = x / (torch.linalg.norm(x) + NS_EPS)
        for _ in range(NS_STEPS):
            gram = torch.mm(x, x.t().contiguous())
            poly = NS_COEFFICIENTS[1] * gram + NS_COEFFICIENTS[2] * torch.mm(gram, gram)
            poly.diagonal().add_(NS_COEFFICIENTS[0])
            x = torch.mm(poly, x)
        out.append(x.t().contiguous() if flip else x)
    return {"out": torch.stack(out)}
