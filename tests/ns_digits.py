"""The digits that newton_schulz keeps: its two-bf16 iterates emulated, and how far a result is from the exact one's
rounding.

A result rounded once to bf16 is 1.5e-3 to 1.7e-3 of the exact result's 2-norm away from it, and an iterate that has
lost its lower halves adds to that only in squares.  From the exact result *rounded to bf16* a result differs where an
error e next to a step u of bf16 carries a value over a boundary: |e| / u of the values, by u each, so by (u |e|)^0.5
in the 2-norm.  A result without errors of its own has a distance of 0, one of the scheme 3e-4 to 5e-4, and one that
leaves out a half or a cross product anywhere 1.2e-3 or more at the sizes of the tests."""

from __future__ import annotations

import torch

from block_oracle import newton_schulz as ns64

COEFFICIENTS = (3.4445, -4.7750, 2.0315)

# What an emulation may leave out: the lower half of an iterate, or a cross product (lo.hi or hi.lo) of a product.
LOSSES = {"A.lo": dict(a=0), "B.lo": dict(b=0), "X.lo": dict(x=0), "hi.lo of X X^T": dict(gram=("lh",)),
          "cross of X X^T": dict(gram=()), "hi.lo of A A": dict(square=("lh",)), "cross of A A": dict(square=()),
          "hi.lo of B X": dict(update=("lh",)), "lo.hi of B X": dict(update=("hl",)), "cross of B X": dict(update=())}


def _halves(v: torch.Tensor, keep: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    hi = v.bfloat16().float()
    return hi, (v - hi).bfloat16().float() * keep


def _product(p, q, cross) -> torch.Tensor:
    r = p[0] @ q[0]
    if "hl" in cross:
        r = r + p[0] @ q[1]
    if "lh" in cross:
        r = r + p[1] @ q[0]
    return r


def emulated(grad: torch.Tensor, steps: int = 5, eps: float = 1e-7, a=1, b=1, x=1, gram=("hl", "lh"),
             square=("hl", "lh"), update=("hl", "lh")) -> torch.Tensor:
    """``newton_schulz(grad)`` of one matrix: X, A and B as two bf16, products without lo.lo, sums in fp32."""
    p, q, r = COEFFICIENTS
    turn = grad.shape[0] > grad.shape[1]
    v = grad.float().t().contiguous() if turn else grad.float()
    v = (v.double() / (torch.linalg.norm(v.double()) + eps)).float()
    X = _halves(v)
    for _ in range(steps):
        A = _halves(_product(X, tuple(t.t().contiguous() for t in X), gram), a)
        B = _halves(r * _product(A, A, square) + q * (A[0] + A[1]), b)
        v = _product(B, X, update) + p * (X[0] + X[1])
        X = _halves(v, x)
    out = v.bfloat16()
    return out.t().contiguous() if turn else out


def distance(out: torch.Tensor, grad: torch.Tensor, steps: int = 5, eps: float = 1e-7) -> float:
    """How far ``out`` is from the 64-bit result rounded to bf16, relative to the result, in the 2-norm."""
    e = ns64(grad, steps, COEFFICIENTS, eps)
    return float((out.double() - e.bfloat16().double()).norm() / e.norm())


def allowed(grad: torch.Tensor, steps: int = 5, eps: float = 1e-7) -> float:
    """The largest distance of a result with all of the scheme's digits: twice the emulation's, four times its error,
    and one value more that is a step of bf16 (2^-7 at most) off, which counts where there are few.

    (The kernels add in another order, which is 2^-24 a sum next to the 2^-18 of the halves.)"""
    return 2 * distance(emulated(grad, steps, eps), grad, steps, eps) + 2.0**-7 / grad.numel() ** 0.5
