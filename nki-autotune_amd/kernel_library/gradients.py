"""The norm over all gradients of a step, and clipping to a largest one, callable on torch device tensors.

* ``grad_norm(grads) -> norm``
* ``clip_grad_norm(grads, max_norm) -> norm, clipped``

bf16, fp16 and fp32 tensors of any sizes, mixed; squares are added in fp64, in an order fixed by the sizes.  Nothing is
copied to the device or waited for: the norm stays there, and so does the factor.  The calls record nothing for torch's
autograd, and warn where it would expect them to (gradients that were recorded themselves, or parameters passed in their
place).  Every call runs HIP kernels (csrc/mi_grad_norm.hpp) on the current torch stream; there is no fallback path.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch

from kernel_library import _lib
from kernel_library._operands import launch, tensor, warn_detached, workspace
from kernel_library.config import _torch_call
from kernel_library.norm import _DTYPES


def _grads(grads: Sequence[torch.Tensor], what: str) -> list[torch.Tensor]:
    if isinstance(grads, torch.Tensor):
        raise TypeError(f"{what} must be a sequence of tensors, got one tensor")
    grads = list(grads)
    if not grads:
        raise ValueError(f"{what} must hold at least one tensor")
    for i, g in enumerate(grads):
        tensor(f"{what}[{i}]", g, _DTYPES, grads[0], f"{what}[0]")
        if not g.is_contiguous():
            raise ValueError(f"{what}[{i}] must be contiguous, got shape {tuple(g.shape)}, strides {g.stride()}")
    return grads


def _run(grads: list[torch.Tensor], outs: list[torch.Tensor] | None, max_norm: float, eps: float) -> torch.Tensor:
    n, device = len(grads), grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=device)
    pointers = ctypes.c_void_p * n
    args = _lib.GradNormArgs(
        ctypes.addressof(ins := pointers(*(g.data_ptr() for g in grads))),
        None if outs is None else ctypes.addressof(outp := pointers(*(o.data_ptr() for o in outs))),
        ctypes.addressof(sizes := (ctypes.c_longlong * n)(*(g.numel() for g in grads))),
        ctypes.addressof(types := (ctypes.c_int * n)(*(_DTYPES[g.dtype] for g in grads))),
        norm.data_ptr(), n, max_norm, eps)
    L = _lib.lib()
    ws, ws_bytes = workspace(device, "clip_grad_norm", L.mi_grad_norm_workspace, ctypes.byref(args))
    launch(device, "clip_grad_norm", L.mi_grad_norm, ctypes.byref(args), ws.data_ptr(), ws_bytes)
    return norm


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """``sqrt(sum g^2)`` over the values of all ``grads``, a 0-dimensional fp32 tensor."""
    done = _torch_call.grad_norm(grads, 0.0, 0.0, None)
    if done is not None:
        return done
    grads = _grads(grads, "grads")
    warn_detached("grad_norm", *grads)
    return _run(grads, None, 0.0, 0.0)


def clip_grad_norm(
    grads: Sequence[torch.Tensor],
    max_norm: float,
    eps: float = 1e-6,
    out: Sequence[torch.Tensor] | None = None,
) -> tuple[torch.Tensor, list[torch.Tensor]]:
    """``(norm, clipped)``: ``clipped[i] = grads[i] * min(1, max_norm / (norm + eps))`` with ``norm = grad_norm(grads)``.

    ``out``: where the clipped gradients go, of their gradients' types and shapes: ``grads`` itself for in place, or
    tensors apart from them; None for new ones.  An infinite norm clips to 0 (and its infinities to NaN), a NaN one to
    NaN, as does an infinite one where ``max_norm`` is infinite too."""
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    if not isinstance(grads, (list, tuple)):
        grads = _grads(grads, "grads")  # (an iterator is read once)
    if out is not None and not isinstance(out, (list, tuple)):
        out = _grads(out, "out")
    # (A C float takes no larger one.)
    most = max_norm if max_norm < 3e38 else math.inf
    done = _torch_call.grad_norm(grads, most, eps, True if out is None else out)
    if done is not None:
        return done if out is None else (done, list(out))
    grads = _grads(grads, "grads")
    outs = [torch.empty_like(g, requires_grad=False) for g in grads] if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"out must hold {len(grads)} tensors, one for each gradient, got {len(outs)}")
    for i, (g, o) in enumerate(zip(grads, _grads(outs, "out"))):
        tensor(f"out[{i}]", o, {g.dtype}, g, f"grads[{i}]")
        if o.shape != g.shape:
            raise ValueError(f"out[{i}] must have grads[{i}]'s shape {tuple(g.shape)}, got {tuple(o.shape)}")
    warn_detached("clip_grad_norm", *grads)
    return _run(grads, list(outs), most, eps), list(outs)
