"""mi_residual_norm_backward with any of its outputs left out: what is wanted is as in the call that wants everything."""

import ctypes
import itertools

import pytest

from test_gpu_residual_norm import TYPES, _check_backward, _inputs

pytestmark = pytest.mark.gpu

OUTPUTS = ("dx", "dweight", "dgate", "dpost_weight")


def _grad(a, dy, dh, hidden, rstd, post_rstd, wanted):
    """The C call with the outputs of ``wanted``; those left out None."""
    import torch

    from kernel_library import _lib

    L, x = _lib.lib(), a["x"]
    D = x.shape[-1]
    like = dict(dx=x, dresidual=hidden, dweight=a["weight"], dgate=a["gate"], dpost_weight=a["post_weight"])
    out = {k: torch.full_like(v, 7.0) if k == "dresidual" or k in wanted else None for k, v in like.items()}
    gate, gates = a["gate"], a["gate"].numel() // D
    dtypes = {torch.bfloat16: _lib.MI_DTYPE_BF16, torch.float16: _lib.MI_DTYPE_F16, torch.float32: _lib.MI_DTYPE_F32}

    def at(t):
        return None if t is None else t.data_ptr()

    args = _lib.ResidualNormGradArgs(
        at(dy), at(dh), at(x), at(hidden), at(a["weight"]), at(gate), at(a["post_weight"]), at(rstd), at(post_rstd),
        *(at(t) for t in out.values()), x.numel() // D, D, D, D, D, gates, D, dtypes[x.dtype],
        hidden.dtype == torch.float32, a["weight"].dtype == torch.float32, gate.dtype == torch.float32, 0.75)
    need = ctypes.c_ulonglong()
    _lib.check_rc(L.mi_residual_norm_backward_workspace(ctypes.byref(args), ctypes.byref(need)), "workspace")
    ws = torch.full((need.value,), 0xFF, dtype=torch.uint8, device=x.device)  # (NaN, where it is read before it is written)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check_rc(L.mi_residual_norm_backward(ctypes.byref(args), at(ws), need.value, stream), "gradient")
    return out


@pytest.mark.parametrize("types", (TYPES[1], TYPES[2], TYPES[4]), ids=lambda t: "-".join(t))
@pytest.mark.parametrize("gate", ("shared", "batch", "full"))
@pytest.mark.parametrize("B,S,D", [(3, 5, 5), (6, 7, 264), (3, 40, 1501), (2, 3, 8192), (2, 3, 9000), (40, 20, 9001)])
def test_outputs_left_out(gpu, B, S, D, gate, types):
    import torch

    import kernel_library as kl

    print(f"residual_norm_backward {B}x{S}x{D} gate {gate} {types}", flush=True)
    a, dy, dh = _inputs(B, S, D, types, gate, True, gpu)
    _, hidden, rstd, post_rstd = kl.residual_norm(scale=0.75, stats=True, **a)
    full = _grad(a, dy, dh, hidden, rstd, post_rstd, OUTPUTS)
    _check_backward(a, 0.75, dy, dh, hidden, rstd, post_rstd,
                    tuple(full[k] for k in ("dx", "dresidual", "dweight", "dgate", "dpost_weight")))
    for n in range(len(OUTPUTS)):
        for wanted in itertools.combinations(OUTPUTS, n):
            got = _grad(a, dy, dh, hidden, rstd, post_rstd, wanted)
            for k, v in got.items():
                if v is None:
                    continue
                if k == "dweight" and gate == "batch" and not {"dgate", "dpost_weight"} & set(wanted):
                    # (No sums by gate: its rows are added in another order.)
                    none = dict.fromkeys(("dx", "dgate", "dpost_weight"))
                    one = dict(full, dweight=v) | none
                    _check_backward(a, 0.75, dy, dh, hidden, rstd, post_rstd,
                                    tuple(one[k] for k in ("dx", "dresidual", "dweight", "dgate", "dpost_weight")))
                else:
                    assert torch.equal(v, full[k]), (wanted, k)
