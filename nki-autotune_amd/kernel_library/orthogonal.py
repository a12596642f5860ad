"""Update matrices orthogonalised by Newton-Schulz products, callable on torch device tensors.

``newton_schulz(grad) -> out`` is the step that the Muon optimiser takes
between its momentum and the weight.  bf16 or fp32 in, bf16 out, one matrix
or a batch of them; the iterates keep 16 bits of mantissa.  The call runs HIP
kernels (csrc/mi_ns.hpp) on the current torch stream; there is no fallback
path.
"""

from __future__ import annotations

import ctypes

import torch

from kernel_library import _lib
from kernel_library._operands import int32, launch, no_overlap, tensor, warn_detached, workspace
from kernel_library.config import _torch_call

_DTYPES = {torch.bfloat16: _lib.MI_DTYPE_BF16, torch.float32: _lib.MI_DTYPE_F32}


def newton_schulz(
    grad: torch.Tensor,
    steps: int = 5,
    coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
    eps: float = 1e-7,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``X = grad / (||grad||_F + eps)``, then ``steps`` times ``A = X X^T; X = a X + (b A + c A A) X``, as bf16.

    ``grad``: ``[m, n]``, or ``[batch, m, n]`` for that many matrices, each by itself; bf16 or fp32, contiguous.
    ``coefficients``: ``(a, b, c)``."""
    if len(coefficients) != 3:
        raise ValueError(f"coefficients must be (a, b, c), got {coefficients!r}")
    done = _torch_call.newton_schulz(grad, steps, *coefficients, eps, out)
    if done is not None:
        return done
    tensor("grad", grad, _DTYPES)
    if grad.dim() not in (2, 3) or not grad.is_contiguous():
        raise ValueError(f"grad must be contiguous, [m, n] or [batch, m, n], got shape {tuple(grad.shape)}")
    if steps < 0:
        raise ValueError(f"steps must be >= 0, got {steps}")
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    batch = grad.shape[0] if grad.dim() == 3 else 1
    m, n = grad.shape[-2:]
    int32(steps=steps, batch=batch, m=m, n=n)
    if out is None:
        out = torch.empty(grad.shape, dtype=torch.bfloat16, device=grad.device)
    else:
        tensor("out", out, (torch.bfloat16,), grad, "grad")
        if out.shape != grad.shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous bf16 tensor of shape {tuple(grad.shape)}")
        no_overlap("out", out, grad=grad)
    warn_detached("newton_schulz", grad)
    args = _lib.NewtonSchulzArgs(grad.data_ptr(), out.data_ptr(), batch, m, n, steps, _DTYPES[grad.dtype], *coefficients,
                                 eps)
    L = _lib.lib()
    ws, ws_bytes = workspace(grad.device, "newton_schulz", L.mi_newton_schulz_workspace, ctypes.byref(args))
    launch(grad.device, "newton_schulz", L.mi_newton_schulz, ctypes.byref(args),
           None if ws is None else ws.data_ptr(), ws_bytes)
    return out
