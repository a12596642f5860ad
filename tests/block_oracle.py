"""Plain 64-bit forms of the training-step operators, for the parity tests (torch, any device)."""

from __future__ import annotations

import math

import torch

ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def half_step(dtype: torch.dtype) -> float:
    """The largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def act(name: str, x: torch.Tensor) -> torch.Tensor:
    if name == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if name == "gelu":
        return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))
    if name == "gelu_tanh":
        # (1 + tanh u) / 2 = 1 / (1 + exp(-2u)), which keeps the digits that 1 + tanh cancels where tanh is near -1.
        return x / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return x


def act_slope(name: str, x: torch.Tensor) -> torch.Tensor:
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-x / math.sqrt(2)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-2 * k * (x + 0.044715 * x**3)))
        return s + x * s * (1 - s) * 2 * k * (1 + 3 * 0.044715 * x * x)
    if name == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s + x * s * (1 - s)
    return torch.ones_like(x)


def matmul_epilogue(lhs, rhs, bias=None, activation="none", residual=None, rhs_transposed=False):
    """(out, pre) in float64."""
    w = rhs.double().t().contiguous() if rhs_transposed else rhs.double()
    pre = lhs.double() @ w
    if bias is not None:
        pre = pre + bias.double()
    out = act(activation, pre)
    return (out if residual is None else out + residual.double()), pre


def matmul_epilogue_tolerance(lhs, rhs, out, bias=None, residual=None, rhs_transposed=False):
    """Largest error of one output rounded to bf16.

    The products are exact in fp32; their sum of K terms, the bias and the residual are rounded at most K + 2 times to
    within 2^-23 (the matrix core may cut where it aligns) of a partial sum that never exceeds the sum of magnitudes.
    No activation is steeper than 1.13, and each is off by at most 2^-19 of its argument (an exponential of argument
    under 100, 2^-24 of it off, and a few more operations).  Then one rounding to bf16."""
    w = rhs.double().abs().t().contiguous() if rhs_transposed else rhs.double().abs()
    mag = lhs.double().abs() @ w
    if bias is not None:
        mag = mag + bias.double().abs()
    tol = 1.13 * (lhs.shape[1] + 2) * 2.0**-23 * mag + 2.0**-19 * mag
    if residual is not None:
        tol = tol + 2.0**-23 * residual.double().abs()
    return tol * (1 + 2.0**-8) + half_step(torch.bfloat16) * out.abs() + 1e-38


def matmul_epilogue_backward(dout, lhs, rhs, activation="none", pre=None, rhs_transposed=False):
    """(dlhs, drhs, dbias, dpre) in float64."""
    dpre = dout.double()
    if activation != "none":
        dpre = dpre * act_slope(activation, pre.double())
    w = rhs.double().t().contiguous() if rhs_transposed else rhs.double()
    dw = lhs.double().t().contiguous() @ dpre
    return dpre @ w.t().contiguous(), dw.t().contiguous() if rhs_transposed else dw, dpre.sum(0), dpre


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) in float64."""
    xd = x.double()
    mean = xd.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((xd - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = (xd - mean) * rstd
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, mean[..., 0], rstd[..., 0]


def layer_norm_backward(dout, x, mean, rstd, weight=None):
    """(dx, dweight, dbias) in float64; column sums over every row."""
    D = x.shape[-1]
    xh = ((x.double() - mean.double()[..., None]) * rstd.double()[..., None]).reshape(-1, D)
    dy = dout.double().reshape(-1, D)
    g = dy if weight is None else dy * weight.double()
    dx = rstd.double().reshape(-1, 1) * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx.reshape(x.shape), (dy * xh).sum(0), dy.sum(0)


def within(actual: torch.Tensor, expected: torch.Tensor, tol) -> None:
    """Every value of ``actual`` within ``tol`` of ``expected`` (not finite where it is not, the same there)."""
    a, e = actual.double(), expected.double()
    assert a.shape == e.shape, (a.shape, e.shape)
    tol = torch.as_tensor(tol, dtype=torch.float64, device=e.device).expand_as(e)
    fine = torch.isfinite(e)
    same = torch.where(torch.isnan(e), torch.isnan(a), a == e)
    ok = torch.where(fine, (a - e).abs() <= tol, same)
    if not bool(ok.all()):
        at = torch.nonzero(~ok)[0].tolist()
        i = tuple(at)
        raise AssertionError(f"{int((~ok).sum())} of {e.numel()} values off; first at {at}: got {float(a[i])!r}, "
                             f"expected {float(e[i])!r} within {float(tol[i])!r}")


def newton_schulz(grad, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """The iterate after ``steps`` steps in float64, of each matrix of a batch."""
    if grad.dim() == 3:
        return torch.stack([newton_schulz(g, steps, coefficients, eps) for g in grad])
    a, b, c = coefficients
    turn = grad.shape[0] > grad.shape[1]
    x = grad.double().t().contiguous() if turn else grad.double()
    x = x / (torch.linalg.norm(x) + eps)
    for _ in range(steps):
        A = x @ x.t().contiguous()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.t().contiguous() if turn else x
