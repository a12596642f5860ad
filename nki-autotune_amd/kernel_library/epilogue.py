"""Products with bias, activation and residual in their epilogue, and their gradients, callable on torch device tensors.

* ``matmul_epilogue(lhs, rhs, bias, activation, residual) -> out``:
  ``out = act(lhs @ rhs + bias) + residual``
* ``matmul_epilogue_backward(dout, lhs, rhs, activation, pre, bias) -> dlhs, drhs, dbias``

bf16 operands and outputs, fp32 accumulation, any sizes; the bias bf16 or
fp32.  ``rhs`` is ``[K, N]`` as in ``matmul_lhs_rhs``, or ``[N, K]`` with
``rhs_transposed`` (``torch.nn.Linear``'s weight).  The calls record nothing
for torch's autograd: the gradient is a call of its own, and the forward call
warns where autograd would expect one.  Every call runs HIP kernels
(csrc/mi_mm_epi.hpp) on the current torch stream; there is no fallback path.
"""

from __future__ import annotations

import ctypes

import torch

from kernel_library import _lib
from kernel_library._operands import int32, launch, no_overlap, tensor, warn_detached, workspace
from kernel_library.config import TileConfig, _torch_call

_ACTIVATIONS = {None: _lib.MI_ACT_NONE, "none": _lib.MI_ACT_NONE, "relu": _lib.MI_ACT_RELU, "gelu": _lib.MI_ACT_GELU,
                "gelu_tanh": _lib.MI_ACT_GELU_TANH, "silu": _lib.MI_ACT_SILU}
_BF16 = (torch.bfloat16,)


def _activation(name: str | None) -> int:
    if name not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(k for k in _ACTIVATIONS if k)} or None, got {name!r}")
    return _ACTIVATIONS[name]


def _operands(lhs: torch.Tensor, rhs: torch.Tensor, rhs_transposed: bool) -> tuple[int, int, int]:
    """(M, N, K) of the product."""
    tensor("lhs", lhs, _BF16)
    tensor("rhs", rhs, _BF16, lhs, "lhs")
    for name, t in (("lhs", lhs), ("rhs", rhs)):
        if t.dim() != 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be 2-D and contiguous (row-major), got shape {tuple(t.shape)}")
    M, K = lhs.shape
    N, K2 = rhs.shape if rhs_transposed else rhs.shape[::-1]
    if K != K2:
        raise ValueError(f"contraction mismatch: lhs has K={K}, rhs has K={K2}")
    int32(M=M, N=N, K=K)
    return M, N, K


def _matrix(name: str, t: torch.Tensor, M: int, N: int, lhs: torch.Tensor) -> None:
    tensor(name, t, _BF16, lhs, "lhs")
    if t.shape != (M, N) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bf16 [{M},{N}] tensor, got shape {tuple(t.shape)}")


def _check_bias(bias: torch.Tensor | None, N: int, lhs: torch.Tensor) -> bool:
    """Checks the bias; whether it is fp32."""
    if bias is None:
        return False
    tensor("bias", bias, (torch.bfloat16, torch.float32), lhs, "lhs")
    if bias.shape != (N,) or not bias.is_contiguous():
        raise ValueError(f"bias must be a contiguous tensor of shape [{N}], got {tuple(bias.shape)}")
    return bias.dtype == torch.float32


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def epilogue_configs() -> list[TileConfig]:
    """The compiled tile configs of ``matmul_epilogue`` (variant 1 reads rhs non-temporally, for few rows)."""
    L, c = _lib.lib(), _lib.MiTileCfg()
    found = []
    for i in range(L.mi_epilogue_num_configs()):
        _lib.check_rc(L.mi_epilogue_config(i, ctypes.byref(c)), "epilogue_configs")
        found.append(TileConfig.from_c(c))
    return found


def matmul_epilogue(
    lhs: torch.Tensor,
    rhs: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    rhs_transposed: bool = False,
    pre: torch.Tensor | None = None,
    cfg: TileConfig | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out[M,N] = act(lhs[M,K] @ rhs[K,N] + bias[N]) + residual[M,N]`` on the GPU (bf16).

    ``activation``: None, "relu", "gelu" (erf), "gelu_tanh" or "silu".  ``pre``, where given, gets ``lhs @ rhs + bias``,
    which the gradient of an activation takes.  ``cfg``: one of ``epilogue_configs()``, any ``split_k`` and
    ``group_m``; None for the library's choice."""
    act = _activation(activation)
    if cfg is None:
        done = _torch_call.matmul_epilogue(lhs, rhs, bias, act, residual, rhs_transposed, pre, out)
        if done is not None:
            return done
    M, N, K = _operands(lhs, rhs, rhs_transposed)
    f32 = _check_bias(bias, N, lhs)
    if residual is not None:
        _matrix("residual", residual, M, N, lhs)
    if pre is not None:
        _matrix("pre", pre, M, N, lhs)
        no_overlap("pre", pre, lhs=lhs, rhs=rhs, bias=bias, residual=residual)
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=lhs.device)
    else:
        _matrix("out", out, M, N, lhs)
        no_overlap("out", out, lhs=lhs, rhs=rhs, bias=bias, residual=residual, pre=pre)
    warn_detached("matmul_epilogue", lhs, rhs, bias, residual)
    args = _lib.EpilogueArgs(lhs.data_ptr(), rhs.data_ptr(), _ptr(bias), _ptr(residual), out.data_ptr(), _ptr(pre), M, N,
                             K, rhs_transposed, act, f32)
    c = None if cfg is None else ctypes.byref(cfg.to_c())
    L = _lib.lib()
    ws, ws_bytes = workspace(lhs.device, "matmul_epilogue", L.mi_matmul_epilogue_workspace, ctypes.byref(args), c)
    launch(lhs.device, "matmul_epilogue", L.mi_matmul_epilogue_bf16, ctypes.byref(args), c, _ptr(ws), ws_bytes)
    return out


def matmul_epilogue_backward(
    dout: torch.Tensor,
    lhs: torch.Tensor,
    rhs: torch.Tensor,
    activation: str | None = None,
    pre: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    rhs_transposed: bool = False,
    need_dlhs: bool = True,
    need_drhs: bool = True,
):
    """``(dlhs, drhs, dbias)`` of ``matmul_epilogue(lhs, rhs, bias, activation, ...)`` for the output's gradient ``dout``.

    ``pre`` is what the forward call wrote, needed for an activation.  ``dbias`` has the bias's type and is None where
    it is (``bias`` is not read); the residual's gradient is ``dout`` itself.  Without ``need_dlhs`` or ``need_drhs``
    that gradient is None and not computed."""
    act = _activation(activation)
    done = _torch_call.matmul_epilogue_backward(dout, lhs, rhs, act, pre, bias, rhs_transposed, need_dlhs, need_drhs)
    if done is not None:
        return done
    M, N, K = _operands(lhs, rhs, rhs_transposed)
    _matrix("dout", dout, M, N, lhs)
    if act != _lib.MI_ACT_NONE:
        if pre is None:
            raise ValueError(f"the gradient of activation {activation!r} needs pre")
        _matrix("pre", pre, M, N, lhs)
    else:
        pre = None
    f32 = _check_bias(bias, N, lhs)
    dlhs = torch.empty_like(lhs) if need_dlhs else None
    drhs = torch.empty_like(rhs) if need_drhs else None
    dbias = None if bias is None else torch.empty_like(bias)
    args = _lib.EpilogueGradArgs(dout.data_ptr(), lhs.data_ptr(), rhs.data_ptr(), _ptr(pre), _ptr(dlhs), _ptr(drhs),
                                 _ptr(dbias), M, N, K, rhs_transposed, act, f32)
    L = _lib.lib()
    ws, ws_bytes = workspace(lhs.device, "matmul_epilogue_backward", L.mi_matmul_epilogue_backward_workspace,
                             ctypes.byref(args))
    launch(lhs.device, "matmul_epilogue_backward", L.mi_matmul_epilogue_backward_bf16, ctypes.byref(args), _ptr(ws),
           ws_bytes)
    return dlhs, drhs, dbias
