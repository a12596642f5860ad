"""Layer norm and its gradients, callable on torch device tensors.

* ``layer_norm(x, weight, bias) -> y`` normalises every row of ``x``
* ``layer_norm_backward(dout, x, mean, rstd, weight, bias) -> dx, dweight, dbias``

bf16, fp16 or fp32 rows of any length; parameters of the rows' type or fp32;
statistics and sums in fp32, each output rounded once.  The calls record
nothing for torch's autograd: the gradient is a call of its own, and the
forward call warns where autograd would expect one.  Every call runs HIP
kernels (csrc/mi_norm.hpp) on the current torch stream; there is no fallback
path.
"""

from __future__ import annotations

import ctypes

import torch

from kernel_library import _lib
from kernel_library._operands import int32, launch, no_overlap, tensor, warn_detached, workspace
from kernel_library.config import _torch_call

_DTYPES = {torch.bfloat16: _lib.MI_DTYPE_BF16, torch.float16: _lib.MI_DTYPE_F16, torch.float32: _lib.MI_DTYPE_F32}


def _rows(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(rows, D, row stride in elements) of ``t`` taken as rows of its last dimension."""
    if t.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")
    D = t.shape[-1]
    if D == 0:
        raise ValueError(f"{name} has rows of no elements, shape {tuple(t.shape)}")
    int32(D=D)
    rows = t.numel() // D
    if t.is_contiguous():
        return rows, D, D
    if t.dim() == 2 and (D == 1 or t.stride(1) == 1):
        return rows, D, t.stride(0)
    raise ValueError(f"{name} must be contiguous, or 2-D with contiguous rows (strides {t.stride()})")


def _params(x: torch.Tensor, D: int, weight: torch.Tensor | None, bias: torch.Tensor | None) -> bool:
    """Checks weight and bias against rows of ``x``; whether they are fp32."""
    kinds = set()
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        tensor(name, t, {x.dtype, torch.float32}, x, "x")
        if t.shape != (D,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of shape [{D}], got {tuple(t.shape)}")
        kinds.add(t.dtype)
    if len(kinds) > 1:
        raise ValueError(f"weight and bias must share a dtype, got {weight.dtype} and {bias.dtype}")
    return torch.float32 in kinds


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    out: torch.Tensor | None = None,
    stats: bool = False,
):
    """``y = (x - mean(x)) / sqrt(var(x) + eps) * weight + bias`` over the last dimension of ``x``.

    With ``stats`` the call returns ``(y, mean, rstd)``, the rows' fp32 statistics that ``layer_norm_backward`` takes
    (of x's shape without its last dimension)."""
    done = _torch_call.layer_norm(x, weight, bias, eps, out, stats)
    if done is not None:
        return done
    tensor("x", x, _DTYPES)
    rows, D, ldx = _rows("x", x)
    f32 = _params(x, D, weight, bias)
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        tensor("out", out, {x.dtype}, x, "x")
        if out.shape != x.shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {x.dtype} tensor of shape {tuple(x.shape)}")
        no_overlap("out", out, x=x, weight=weight, bias=bias)
    warn_detached("layer_norm", x, weight, bias)
    mean = rstd = None
    if stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    if rows:
        args = _lib.LayerNormArgs(x.data_ptr(), _ptr(weight), _ptr(bias), out.data_ptr(), _ptr(mean), _ptr(rstd), rows,
                                  ldx, D, _DTYPES[x.dtype], f32, eps)
        launch(x.device, "layer_norm", _lib.lib().mi_layer_norm, ctypes.byref(args))
    return (out, mean, rstd) if stats else out


def layer_norm_backward(
    dout: torch.Tensor,
    x: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    need_dx: bool = True,
):
    """``(dx, dweight, dbias)`` of ``layer_norm(x, weight, bias)`` for the output's gradient ``dout``.

    ``mean`` and ``rstd`` are what the forward call returned with ``stats``.  ``dweight`` and ``dbias`` have their
    parameter's type and are None where it is (``bias`` is not read); ``dx`` is None without ``need_dx``."""
    done = _torch_call.layer_norm_backward(dout, x, mean, rstd, weight, bias, need_dx)
    if done is not None:
        return done
    tensor("x", x, _DTYPES)
    rows, D, ldx = _rows("x", x)
    tensor("dout", dout, {x.dtype}, x, "x")
    if dout.shape != x.shape:
        raise ValueError(f"dout must have x's shape {tuple(x.shape)}, got {tuple(dout.shape)}")
    _, _, lddout = _rows("dout", dout)
    for name, t in (("mean", mean), ("rstd", rstd)):
        tensor(name, t, {torch.float32}, x, "x")
        if t.shape != x.shape[:-1] or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of shape {tuple(x.shape[:-1])}, got {tuple(t.shape)}")
    f32 = _params(x, D, weight, bias)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
    dweight = None if weight is None else torch.empty_like(weight)
    dbias = None if bias is None else torch.empty_like(bias)
    args = _lib.LayerNormGradArgs(dout.data_ptr(), x.data_ptr(), _ptr(weight), mean.data_ptr(), rstd.data_ptr(), _ptr(dx),
                                  _ptr(dweight), _ptr(dbias), rows, lddout, ldx, D, _DTYPES[x.dtype], f32)
    L = _lib.lib()
    ws, ws_bytes = workspace(x.device, "layer_norm_backward", L.mi_layer_norm_backward_workspace, ctypes.byref(args))
    launch(x.device, "layer_norm_backward", L.mi_layer_norm_backward, ctypes.byref(args), _ptr(ws), ws_bytes)
    return dx, dweight, dbias
