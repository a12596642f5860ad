"""Products in 8-bit floating point with a scale for each block of 128, their operands and gradients, callable on torch
device tensors.

* ``quantize_fp8(x) -> q, scale``: a matrix in e4m3 or e5m2 with a scale for each 1 x 128 or 128 x 128 values, and of
  the same reading its transpose
* ``matmul_fp8(lhs, lhs_scale, rhs, rhs_scale) -> out``: ``out[M, N] = lhs[M, K] @ rhs[N, K].T`` of what they stand for
* ``matmul_fp8_backward(dout, lhs_t, ..., rhs_t, ...) -> dlhs, drhs``

Both operands are K-contiguous, as the 8-bit matrix instructions take them: ``rhs`` is ``[N, K]``, as
``torch.nn.Linear`` has its weight.  Scales are fp32, or powers of two (``torch.float8_e8m0fnu``), which the matrix
instructions apply themselves.  The calls record nothing for torch's autograd: the gradient is a call of its own, and
the others warn where autograd would expect one.  Every call runs HIP kernels (csrc/mi_quant.hpp, csrc/mi_mm_fp8.hpp)
on the current torch stream; there is no fallback path.
"""

from __future__ import annotations

import ctypes

import torch

from kernel_library import _lib
from kernel_library._operands import int32, launch, no_overlap, tensor, warn_detached, workspace
from kernel_library.config import TileConfig, _torch_call
from kernel_library.norm import _DTYPES, _ptr

BLOCK = 128
_FP8 = {torch.float8_e4m3fn: _lib.MI_FP8_E4M3, torch.float8_e5m2: _lib.MI_FP8_E5M2}
_E4M3 = (torch.float8_e4m3fn,)
_SCALES = (torch.float32, torch.float8_e8m0fnu)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _up16(n: int) -> int:
    return -(-n // 16) * 16


def _member(name: str, value: object, allowed) -> None:
    if value not in allowed:
        raise ValueError(f"{name} must be one of {tuple(allowed)}, got {value!r}")


def _matrix(name: str, t: torch.Tensor, dtypes, ref: torch.Tensor | None = None, ref_name: str = "") -> int:
    """Checks a matrix of consecutive values in each row; its row stride."""
    tensor(name, t, dtypes, ref, ref_name)
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be 2-D with contiguous rows, got shape {tuple(t.shape)}, strides {t.stride()}")
    int32(rows=t.shape[0], columns=t.shape[1])
    return t.stride(0)


def _scale(name: str, s: torch.Tensor, of: str, t: torch.Tensor, square: bool) -> bool:
    """Checks the scales of ``t``; whether they are for 128 x 128 values (``square``: they may be)."""
    tensor(name, s, _SCALES, t, of)
    rows, blocks = t.shape[0], _blocks(t.shape[1])
    if s.dim() == 2 and s.shape[1] == blocks:
        if s.shape[0] == rows:
            return False
        if square and s.shape[0] == _blocks(rows):
            return True
    allowed = f"[{rows}, {blocks}]" + (f" or [{_blocks(rows)}, {blocks}]" if square else "")
    raise ValueError(f"{name} must have shape {allowed} for {of} {tuple(t.shape)}, got {tuple(s.shape)}")


def _rows(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Rows of 8-bit values that start on 16 bytes."""
    t = torch.empty((rows, _up16(cols)), dtype=dtype, device=device)
    return t[:, :cols] if cols % 16 else t


def _scales(rows: int, cols: int, square: bool, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """The scales of a [rows, cols] matrix, those of 1 x 128 values with the rows consecutive in memory."""
    if square:
        return torch.empty((_blocks(rows), _blocks(cols)), dtype=dtype, device=device)
    return torch.empty((_blocks(cols), rows), dtype=dtype, device=device).t()


def quantize_fp8(
    x: torch.Tensor,
    block: tuple[int, int] = (1, BLOCK),
    dtype: torch.dtype = torch.float8_e4m3fn,
    scale_dtype: torch.dtype = torch.float32,
    transposed: bool = False,
):
    """``x [M, K]`` (bf16, fp16 or fp32) as ``(q, scale)``: ``q [M, K]`` of ``dtype`` and a scale for each ``block`` of it.

    ``block``: ``(1, 128)``, ``scale [M, ceil(K / 128)]``, or ``(128, 128)``, ``scale [ceil(M / 128), ceil(K / 128)]``.
    ``scale_dtype`` fp32: the largest magnitude over the type's largest value, at least 2^-100; ``float8_e8m0fnu``: the
    least power of two from there on.  ``q`` is ``x / scale``, rounded to fp32 and then to ``dtype``.  A block that holds
    an infinity or a NaN is NaN throughout.  With ``transposed`` the call returns ``(q, scale, q_t, scale_t)``, the last
    two of ``x.T [K, M]``, whose 1 x 128 blocks are 128 rows of ``x``.  Rows of ``q`` start on 16 bytes: where K is no
    multiple of 16, ``q`` is a view of wider rows, filled with zeros."""
    if tuple(block) not in ((1, BLOCK), (BLOCK, BLOCK)):
        raise ValueError(f"block must be (1, {BLOCK}) or ({BLOCK}, {BLOCK}), got {block}")
    _member("dtype", dtype, _FP8)
    _member("scale_dtype", scale_dtype, _SCALES)
    square, e8m0 = block[0] != 1, scale_dtype != torch.float32
    done = _torch_call.quantize_fp8(x, square, _FP8[dtype], e8m0, transposed)
    if done is not None:
        return done
    ldx = _matrix("x", x, _DTYPES)
    warn_detached("quantize_fp8", x)
    M, K = x.shape
    q, scale = _rows(M, K, dtype, x.device), _scales(M, K, square, scale_dtype, x.device)
    q_t = scale_t = None
    if transposed:
        q_t, scale_t = _rows(K, M, dtype, x.device), _scales(K, M, square, scale_dtype, x.device)
    if M and K:
        args = _lib.QuantizeFp8Args(x.data_ptr(), q.data_ptr(), scale.data_ptr(), _ptr(q_t), _ptr(scale_t), ldx, _up16(K),
                                    _up16(M), M, K, _DTYPES[x.dtype], _FP8[dtype], e8m0, square)
        launch(x.device, "quantize_fp8", _lib.lib().mi_quantize_fp8, ctypes.byref(args))
    return (q, scale, q_t, scale_t) if transposed else (q, scale)


def fp8_configs() -> list[TileConfig]:
    """The compiled tile configs of ``matmul_fp8`` (variant 1 reads rhs non-temporally, for few rows)."""
    L, c = _lib.lib(), _lib.MiTileCfg()
    found = []
    for i in range(L.mi_fp8_num_configs()):
        _lib.check_rc(L.mi_fp8_config(i, ctypes.byref(c)), "fp8_configs")
        found.append(TileConfig.from_c(c))
    return found


def matmul_fp8(
    lhs: torch.Tensor,
    lhs_scale: torch.Tensor,
    rhs: torch.Tensor,
    rhs_scale: torch.Tensor,
    cfg: TileConfig | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out[M, N] = (lhs * lhs_scale)[M, K] @ (rhs * rhs_scale)[N, K].T``, each scale for 128 values along K.

    ``lhs``: e4m3 or e5m2, ``lhs_scale [M, ceil(K / 128)]``; ``rhs``: e4m3, ``rhs_scale [N, ceil(K / 128)]`` or, for 128
    rows at a time, ``[ceil(N / 128), ceil(K / 128)]``; both scales fp32 or both ``float8_e8m0fnu``, of any strides (those
    of ``quantize_fp8`` are read fastest); ``out``: bf16.  ``cfg``: one of ``fp8_configs()``, any
    ``split_k`` and ``group_m``; None for the library's choice.

    The values' products are exact.  The matrix instructions add 8 consecutive ones at a time and drop what lies below
    2^-13 of the largest (about 1e-5 of a result of normally distributed values, where the rounding to bf16 is up to 2^-8);
    these sums are added in fp32.  The product of two fp32 scales is rounded to fp32 too: it has to be finite, and below
    2^-126 it is a multiple of 2^-149."""
    if cfg is None:
        done = _torch_call.matmul_fp8(lhs, lhs_scale, rhs, rhs_scale, out)
        if done is not None:
            return done
    ldl = _matrix("lhs", lhs, _FP8)
    ldr = _matrix("rhs", rhs, _E4M3, lhs, "lhs")
    (M, K), N = lhs.shape, rhs.shape[0]
    if rhs.shape[1] != K:
        raise ValueError(f"contraction mismatch: lhs has K={K}, rhs has K={rhs.shape[1]}")
    _scale("lhs_scale", lhs_scale, "lhs", lhs, False)
    square = _scale("rhs_scale", rhs_scale, "rhs", rhs, True)
    if lhs_scale.dtype != rhs_scale.dtype:
        raise ValueError(f"lhs_scale and rhs_scale must share a dtype, got {lhs_scale.dtype} and {rhs_scale.dtype}")
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=lhs.device)
    else:
        tensor("out", out, (torch.bfloat16,), lhs, "lhs")
        if out.shape != (M, N) or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous bf16 [{M},{N}] tensor, got shape {tuple(out.shape)}")
        no_overlap("out", out, lhs=lhs, lhs_scale=lhs_scale, rhs=rhs, rhs_scale=rhs_scale)
    warn_detached("matmul_fp8", lhs, lhs_scale, rhs, rhs_scale)
    args = _lib.MatmulFp8Args(lhs.data_ptr(), rhs.data_ptr(), lhs_scale.data_ptr(), rhs_scale.data_ptr(), out.data_ptr(),
                              ldl, ldr, *lhs_scale.stride(), *rhs_scale.stride(), M, N, K, _FP8[lhs.dtype],
                              lhs_scale.dtype != torch.float32, square)
    c = None if cfg is None else ctypes.byref(cfg.to_c())
    L = _lib.lib()
    ws, ws_bytes = workspace(lhs.device, "matmul_fp8", L.mi_matmul_fp8_workspace, ctypes.byref(args), c)
    launch(lhs.device, "matmul_fp8", L.mi_matmul_fp8, ctypes.byref(args), c, _ptr(ws), ws_bytes)
    return out


def matmul_fp8_backward(
    dout: torch.Tensor,
    lhs_t: torch.Tensor | None,
    lhs_t_scale: torch.Tensor | None,
    rhs_t: torch.Tensor | None,
    rhs_t_scale: torch.Tensor | None,
    dtype: torch.dtype = torch.float8_e4m3fn,
    need_dlhs: bool = True,
    need_drhs: bool = True,
):
    """``(dlhs [M, K], drhs [N, K])``, bf16, of ``matmul_fp8`` for the output's gradient ``dout [M, N]`` (bf16).

    ``lhs_t [K, M]`` and ``rhs_t [K, N]`` are the operands' transposes, e4m3, with scales along M and N:
    ``quantize_fp8(..., transposed=True)`` gives them (``rhs_t_scale`` for 1 x 128 or 128 x 128 values).  ``dout`` is
    brought to ``dtype`` inside, in blocks of 1 x 128 along N for ``dlhs`` and along M for ``drhs``, with scales of the
    operands' type.  Without ``need_dlhs`` (``need_drhs``) that gradient is
    None, and ``rhs_t`` (``lhs_t``) is not read."""
    _member("dtype", dtype, _FP8)
    if need_dlhs and need_drhs:
        done = _torch_call.matmul_fp8_backward(dout, lhs_t, lhs_t_scale, rhs_t, rhs_t_scale, _FP8[dtype])
        if done is not None:
            return done
    lddout = _matrix("dout", dout, (torch.bfloat16,))
    M, N = dout.shape
    if not need_dlhs and not need_drhs:
        return None, None
    K, kinds, square, ldl, ldr, strides = None, set(), False, 0, 0, {"lhs_t": (0, 0), "rhs_t": (0, 0)}
    for name, t, s, need, cols in (("lhs_t", lhs_t, lhs_t_scale, need_drhs, M), ("rhs_t", rhs_t, rhs_t_scale, need_dlhs, N)):
        if not need:
            continue
        ld = _matrix(name, t, _E4M3, dout, "dout")
        if t.shape[1] != cols or (K is not None and t.shape[0] != K):
            raise ValueError(f"{name} must have shape [{'K' if K is None else K}, {cols}], got {tuple(t.shape)}")
        K = t.shape[0]
        whole = _scale(f"{name}_scale", s, name, t, name == "rhs_t")
        kinds.add(s.dtype)
        strides[name] = s.stride()
        if name == "lhs_t":
            ldl = ld
        else:
            ldr, square = ld, whole
    if len(kinds) > 1:
        raise ValueError(f"lhs_t_scale and rhs_t_scale must share a dtype, got {lhs_t_scale.dtype} and {rhs_t_scale.dtype}")
    dlhs = torch.empty((M, K), dtype=torch.bfloat16, device=dout.device) if need_dlhs else None
    drhs = torch.empty((N, K), dtype=torch.bfloat16, device=dout.device) if need_drhs else None
    args = _lib.MatmulFp8GradArgs(
        dout.data_ptr(), _ptr(lhs_t if need_drhs else None), _ptr(lhs_t_scale if need_drhs else None),
        _ptr(rhs_t if need_dlhs else None), _ptr(rhs_t_scale if need_dlhs else None), _ptr(dlhs), _ptr(drhs), lddout, ldl,
        ldr, *strides["lhs_t"], *strides["rhs_t"], M, N, K, _FP8[dtype], torch.float32 not in kinds, square)
    L = _lib.lib()
    ws, ws_bytes = workspace(dout.device, "matmul_fp8_backward", L.mi_matmul_fp8_backward_workspace, ctypes.byref(args))
    launch(dout.device, "matmul_fp8_backward", L.mi_matmul_fp8_backward, ctypes.byref(args), _ptr(ws), ws_bytes)
    return dlhs, drhs
