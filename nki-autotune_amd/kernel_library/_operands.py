"""Argument checks, workspaces and launches shared by the operators that take argument structures."""

from __future__ import annotations

import ctypes
import os
import warnings
from collections.abc import Callable, Container

import torch

from kernel_library import _lib
from kernel_library.config import _torch_call

_ENTRY_POINTS = ("mi_layer_norm", "mi_layer_norm_backward_workspace", "mi_layer_norm_backward",
                 "mi_matmul_epilogue_workspace", "mi_matmul_epilogue_bf16", "mi_matmul_epilogue_backward_workspace",
                 "mi_matmul_epilogue_backward_bf16", "mi_newton_schulz_workspace", "mi_newton_schulz")


def tensor(name: str, t: object, dtypes: Container[torch.dtype], ref: torch.Tensor | None = None,
           ref_name: str = "") -> None:
    """``t`` is a tensor of one of ``dtypes`` on a HIP device (``ref``'s, where given)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor on a HIP device, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on a HIP device (got {t.device})")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} dtype {t.dtype} not in {tuple(dtypes)}")
    if t.is_neg():
        raise ValueError(f"{name} is a negated view: its memory holds other values (resolve_neg() first)")
    if ref is not None and t.device != ref.device:
        raise ValueError(f"{name} is on {t.device}, {ref_name} on {ref.device}: all operands must share a device")


def int32(**values: int) -> None:
    """The values that a C int takes (ctypes would cut them to it)."""
    for name, v in values.items():
        if not -2**31 <= v < 2**31:
            raise ValueError(f"{name}={v} does not fit 32 bits")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The first byte of ``t`` and the one past its last."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def no_overlap(name: str, out: torch.Tensor, **others: torch.Tensor | None) -> None:
    """``out`` shares no bytes with another operand: the kernels read those while they write ``out``."""
    o0, o1 = _span(out)
    for other, t in others.items():
        if t is None:
            continue
        t0, t1 = _span(t)
        if t0 < o1 and o0 < t1:
            raise ValueError(f"{name} overlaps {other}: an output must not alias another operand")


def warn_detached(what: str, *operands: torch.Tensor | None) -> None:
    """Warns (at the caller of the operator that calls this) where autograd records and an operand requires a gradient:
    the result will not."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        warnings.warn(f"{what} records nothing for autograd, and an operand requires a gradient: it will not reach it "
                      f"through this result. Call {what} under torch.no_grad() and take the gradients from the "
                      "operator's own call.", UserWarning, stacklevel=3)


def _on(device: torch.device, fn: Callable, *args) -> int:
    """``fn(*args)`` with ``device`` as the current one: the library plans for, and launches on, that."""
    if device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def workspace(device: torch.device, what: str, query: Callable, *args) -> tuple[torch.Tensor | None, int]:
    """The workspace that a call needs, and its bytes: from torch's allocator on the current stream, so that calls on
    several streams, and graphs, have one each."""
    need = ctypes.c_ulonglong()
    _lib.check_rc(_on(device, query, *args, ctypes.byref(need)), what)
    if not need.value:
        return None, 0
    return torch.empty(need.value, dtype=torch.uint8, device=device), need.value


def launch(device: torch.device, what: str, fn: Callable, *args) -> None:
    """``fn(*args, stream)`` on the current stream of ``device``; the native calls learn of the library that ran it."""
    stream = torch.cuda.current_stream(device).cuda_stream
    _lib.check_rc(_on(device, fn, *args, stream), what)
    if not _torch_call.knows_operators():
        L = _lib.lib()
        _torch_call.bind_operators(os.environ.get("MI_KERNELS_LIB", ""),
                                   *(ctypes.cast(getattr(L, f), ctypes.c_void_p).value for f in _ENTRY_POINTS),
                                   _lib.check_rc)
