"""MI355X (gfx950) kernel_library: hand-written HIP kernels behind a C ABI.

Public kernels (torch device tensors in, torch device tensor out):

* :func:`matmul_lhsT_rhs` -- ``lhs_T[K,M].T @ rhs[K,N]``, bf16 or fp32
* :func:`matmul_lhs_rhs` -- ``lhs[M,K] @ rhs[K,N]``, bf16
* :func:`rmsnorm_matmul` -- ``rmsnorm(lhs) * gamma @ rhs``, bf16
* :func:`matmul_epilogue` -- ``act(lhs @ rhs + bias) + residual``, bf16, and :func:`matmul_epilogue_backward`
* :func:`newton_schulz` -- an update matrix orthogonalised (the Muon optimiser's step), bf16 or fp32
* :func:`layer_norm` -- bf16, fp16 or fp32, and :func:`layer_norm_backward`

plus the reference names ``matmul_lhsT_rhs_nkigym``, ``matmul_lhs_rhs_nkigym`` and
``rmsnorm_matmul_online``, the tile search space (:class:`TileConfig`), and
:func:`release_workspace` (returns the cached split-K workspace memory).
"""

from kernel_library.config import (
    TileConfig,
    baseline_grid,
    check,
    compiled_configs,
    default_config,
    legal_configs,
)
from kernel_library.epilogue import epilogue_configs, matmul_epilogue, matmul_epilogue_backward
from kernel_library.norm import layer_norm, layer_norm_backward
from kernel_library.orthogonal import newton_schulz
from kernel_library.ops import (
    EPS,
    matmul_lhs_rhs,
    matmul_lhs_rhs_nkigym,
    matmul_lhsT_rhs,
    matmul_lhsT_rhs_nkigym,
    release_workspace,
    rmsnorm_matmul,
    rmsnorm_matmul_online,
)

__all__ = [
    "EPS",
    "TileConfig",
    "baseline_grid",
    "check",
    "compiled_configs",
    "default_config",
    "epilogue_configs",
    "layer_norm",
    "layer_norm_backward",
    "legal_configs",
    "matmul_epilogue",
    "matmul_epilogue_backward",
    "matmul_lhs_rhs",
    "newton_schulz",
    "matmul_lhs_rhs_nkigym",
    "matmul_lhsT_rhs",
    "matmul_lhsT_rhs_nkigym",
    "release_workspace",
    "rmsnorm_matmul",
    "rmsnorm_matmul_online",
]
