"""What layer_norm, matmul_epilogue, newton_schulz and the gradients refuse: the C ABI's codes, before any launch (no
call here touches a GPU), and the Python checks on tensors that are not on one."""

from __future__ import annotations

import ctypes

import pytest
import torch

import kernel_library as kl
from kernel_library import _lib

P = 1 << 40  # an address that nothing is at: refused calls do not use it
GIB = 1 << 30


def _at(i: int) -> int:
    return P + i * 64 * GIB


def _code(fn, args, *rest) -> int:
    rc = fn(ctypes.byref(args), *rest)
    assert rc == 0 or _lib.last_error(), "a refusal says why"
    return rc


def _ln(**kw):
    a = dict(x=_at(0), weight=_at(1), bias=_at(2), y=_at(3), mean=_at(4), rstd=_at(5), rows=8, ldx=64, D=64,
             dtype=_lib.MI_DTYPE_BF16, params_f32=0, eps=1e-5)
    return _lib.LayerNormArgs(**(a | kw))


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.MI_E_ARGS),
    (dict(D=0), _lib.MI_E_ARGS),
    (dict(D=-4), _lib.MI_E_ARGS),
    (dict(D=GIB + 1), _lib.MI_E_RANGE),
    (dict(ldx=-64), _lib.MI_E_ARGS),
    (dict(dtype=3), _lib.MI_E_ARGS),
    (dict(dtype=-1), _lib.MI_E_ARGS),
    (dict(eps=-1e-5), _lib.MI_E_ARGS),
    (dict(eps=float("nan")), _lib.MI_E_ARGS),
    (dict(eps=float("inf")), _lib.MI_E_ARGS),
    (dict(x=None), _lib.MI_E_ARGS),
    (dict(y=None), _lib.MI_E_ARGS),
    (dict(x=_at(0) + 1), _lib.MI_E_ALIGN),
    (dict(weight=_at(1) + 2, params_f32=1), _lib.MI_E_ALIGN),
    (dict(mean=_at(4) + 2), _lib.MI_E_ALIGN),
    (dict(y=_at(0)), _lib.MI_E_ARGS),
    (dict(y=_at(0) + 2 * 8 * 64 - 2), _lib.MI_E_ARGS),
    (dict(y=_at(0) - 2), _lib.MI_E_ARGS),
    (dict(y=_at(1) + 2), _lib.MI_E_ARGS),
    (dict(y=_at(5)), _lib.MI_E_ARGS),
    (dict(mean=_at(0)), _lib.MI_E_ARGS),
    (dict(rstd=_at(4)), _lib.MI_E_ARGS),
    (dict(rows=0, x=None, y=None), _lib.MI_OK),
])
def test_layer_norm(kw, code):
    assert _code(_lib.lib().mi_layer_norm, _ln(**kw), None) == code


def _ln_bwd(**kw):
    a = dict(dout=_at(0), x=_at(1), weight=_at(2), mean=_at(3), rstd=_at(4), dx=_at(5), dweight=_at(6), dbias=_at(7),
             rows=8, lddout=64, ldx=64, D=64, dtype=_lib.MI_DTYPE_BF16, params_f32=0)
    return _lib.LayerNormGradArgs(**(a | kw))


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.MI_E_ARGS),
    (dict(D=0), _lib.MI_E_ARGS),
    (dict(dtype=7), _lib.MI_E_ARGS),
    (dict(lddout=-1), _lib.MI_E_ARGS),
    (dict(x=None), _lib.MI_E_ARGS),
    (dict(rstd=None), _lib.MI_E_ARGS),
    (dict(dout=_at(0) + 1), _lib.MI_E_ALIGN),
    (dict(dweight=_at(6) + 2, params_f32=1), _lib.MI_E_ALIGN),
    (dict(dx=_at(1)), _lib.MI_E_ARGS),
    (dict(dx=_at(0) + 64), _lib.MI_E_ARGS),
    (dict(dbias=_at(6)), _lib.MI_E_ARGS),
    (dict(dweight=_at(2)), _lib.MI_E_ARGS),
    (dict(dx=_at(9)), _lib.MI_E_ARGS),  # the workspace
    (dict(dx=None, dweight=None, dbias=None), _lib.MI_OK),
    (dict(D=(1 << 28) + 1), _lib.MI_E_RANGE),
])
def test_layer_norm_backward(kw, code):
    L = _lib.lib()
    assert _code(L.mi_layer_norm_backward, _ln_bwd(**kw), _at(9), GIB, None) == code


def test_layer_norm_backward_workspace():
    L = _lib.lib()
    need = ctypes.c_ulonglong()
    assert _code(L.mi_layer_norm_backward_workspace, _ln_bwd(), ctypes.byref(need)) == 0 and need.value > 0
    short = need.value - 1
    assert _code(L.mi_layer_norm_backward, _ln_bwd(), _at(9), short, None) == _lib.MI_E_ARGS
    assert _code(L.mi_layer_norm_backward, _ln_bwd(), None, 0, None) == _lib.MI_E_ARGS
    assert _code(L.mi_layer_norm_backward, _ln_bwd(), _at(9) + 8, GIB, None) == _lib.MI_E_ARGS
    for kw in (dict(dweight=None, dbias=None), dict(rows=0)):
        assert _code(L.mi_layer_norm_backward_workspace, _ln_bwd(**kw), ctypes.byref(need)) == 0 and need.value == 0
    assert L.mi_layer_norm_backward_workspace(None, ctypes.byref(need)) == _lib.MI_E_ARGS
    assert L.mi_layer_norm(None, None) == _lib.MI_E_ARGS


def _mm(**kw):
    a = dict(lhs=_at(0), rhs=_at(1), bias=_at(2), residual=_at(3), out=_at(4), pre=_at(5), M=64, N=64, K=64,
             rhs_transposed=0, activation=0, bias_f32=0)
    return _lib.EpilogueArgs(**(a | kw))


BIG = 2**31 - 1


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), _lib.MI_E_ARGS),
    (dict(K=-8), _lib.MI_E_ARGS),
    (dict(activation=5), _lib.MI_E_ARGS),
    (dict(activation=-1), _lib.MI_E_ARGS),
    (dict(M=1 << 16, K=1 << 16), _lib.MI_E_RANGE),
    (dict(N=1 << 16, K=1 << 16), _lib.MI_E_RANGE),
    (dict(M=BIG, N=BIG, K=0), _lib.MI_E_RANGE),
    (dict(M=1, N=BIG, K=1), _lib.MI_E_RANGE),
    (dict(M=1, N=1, K=BIG), _lib.MI_E_RANGE),
    (dict(M=BIG - (1 << 20) + 1, N=1, K=0), _lib.MI_E_RANGE),
    (dict(lhs=None), _lib.MI_E_ARGS),
    (dict(out=None), _lib.MI_E_ARGS),
    (dict(lhs=_at(0) + 1), _lib.MI_E_ALIGN),
    (dict(bias=_at(2) + 2, bias_f32=1), _lib.MI_E_ALIGN),
    (dict(pre=_at(5) + 1), _lib.MI_E_ALIGN),
    (dict(out=_at(3)), _lib.MI_E_ARGS),
    (dict(out=_at(0) + 64 * 64 * 2 - 2), _lib.MI_E_ARGS),
    (dict(pre=_at(4)), _lib.MI_E_ARGS),
    (dict(pre=_at(2)), _lib.MI_E_ARGS),
    (dict(out=_at(9), M=512, K=63), _lib.MI_E_ARGS),  # the workspace
    (dict(M=0, lhs=None, out=None), _lib.MI_OK),
    (dict(N=0, rhs=None, out=None), _lib.MI_OK),
])
def test_matmul_epilogue(kw, code):
    assert _code(_lib.lib().mi_matmul_epilogue_bf16, _mm(**kw), None, _at(9), 8 * GIB, None) == code


@pytest.mark.parametrize("cfg,code", [
    (kl.TileConfig(128, 128, 64, 4, 4, split_k=0), _lib.MI_E_SPLIT),
    (kl.TileConfig(128, 128, 64, 4, 4, split_k=17), _lib.MI_E_SPLIT),
    (kl.TileConfig(128, 128, 64, 4, 4, split_k=2), _lib.MI_E_SPLIT),  # one K tile
    (kl.TileConfig(128, 128, 64, 4, 4, group_m=-1), _lib.MI_E_ARGS),
    (kl.TileConfig(128, 128, 32, 4, 4), _lib.MI_E_NO_INSTANCE),
    (kl.TileConfig(512, 512, 64, 8, 2), _lib.MI_E_NO_INSTANCE),
])
def test_matmul_epilogue_configs(cfg, code):
    L, c = _lib.lib(), cfg.to_c()
    assert _code(L.mi_matmul_epilogue_bf16, _mm(), ctypes.byref(c), _at(9), GIB, None) == code
    need = ctypes.c_ulonglong()
    assert _code(L.mi_matmul_epilogue_workspace, _mm(), ctypes.byref(c), ctypes.byref(need)) == code
    assert need.value == 0


def test_matmul_epilogue_wide_outputs_are_not_split():
    L, need = _lib.lib(), ctypes.c_ulonglong()
    wide = _mm(M=1, N=(1 << 20) + 8, K=1024)
    c = kl.TileConfig(128, 128, 64, 4, 4, split_k=2).to_c()
    assert _code(L.mi_matmul_epilogue_workspace, wide, ctypes.byref(c), ctypes.byref(need)) == _lib.MI_E_SPLIT
    assert _code(L.mi_matmul_epilogue_workspace, wide, None, ctypes.byref(need)) == 0 and need.value == 0


def test_matmul_epilogue_workspace():
    L, need = _lib.lib(), ctypes.c_ulonglong()
    for kw, copies in ((dict(), 0), (dict(K=63), 512), (dict(K=63, rhs_transposed=1), 512 + 64), (dict(N=63), 64),
                       (dict(N=63, rhs_transposed=1), 0), (dict(lhs=_at(0) + 2), 512), (dict(rhs=_at(1) + 8), 64),
                       (dict(K=0), 0), (dict(M=0), 0)):
        assert _code(L.mi_matmul_epilogue_workspace, _mm(**(dict(M=512) | kw)), None, ctypes.byref(need)) == 0
        assert need.value == copies * 64 * 2, kw
    assert _code(L.mi_matmul_epilogue_bf16, _mm(M=512, K=63), None, None, 0, None) == _lib.MI_E_ARGS
    assert _code(L.mi_matmul_epilogue_bf16, _mm(M=512, K=63), None, _at(9) + 2, GIB, None) == _lib.MI_E_ARGS
    # Few rows: no copies, unless a config asks for the kernels that need them or there is no whole 16-byte piece.
    c = kl.TileConfig(64, 64, 64, 4, 2).to_c()
    for kw, cfg, copies in ((dict(K=63), None, 0), (dict(N=63), None, 0), (dict(K=63), ctypes.byref(c), 64),
                            (dict(K=7), None, 8), (dict(N=7), None, 8)):
        assert _code(L.mi_matmul_epilogue_workspace, _mm(**kw), cfg, ctypes.byref(need)) == 0
        assert need.value == copies * 64 * 2, kw
    assert L.mi_matmul_epilogue_workspace(None, None, ctypes.byref(need)) == _lib.MI_E_ARGS
    assert L.mi_matmul_epilogue_bf16(None, None, None, 0, None) == _lib.MI_E_ARGS


def _mm_bwd(**kw):
    a = dict(dout=_at(0), lhs=_at(1), rhs=_at(2), pre=_at(3), dlhs=_at(4), drhs=_at(5), dbias=_at(6), M=64, N=64, K=64,
             rhs_transposed=0, activation=_lib.MI_ACT_GELU, bias_f32=0)
    return _lib.EpilogueGradArgs(**(a | kw))


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), _lib.MI_E_ARGS),
    (dict(activation=9), _lib.MI_E_ARGS),
    (dict(dout=None), _lib.MI_E_ARGS),
    (dict(pre=None), _lib.MI_E_ARGS),
    (dict(rhs=None), _lib.MI_E_ARGS),
    (dict(lhs=None), _lib.MI_E_ARGS),
    (dict(M=1 << 20, N=1 << 14), _lib.MI_E_RANGE),
    (dict(M=1 << 20, N=1 << 14, dlhs=None), _lib.MI_E_RANGE),
    (dict(M=BIG - (1 << 20) + 1, N=1, K=0), _lib.MI_E_RANGE),
    (dict(M=1, N=(1 << 28) + 1, K=0), _lib.MI_E_RANGE),
    (dict(dout=_at(0) + 1), _lib.MI_E_ALIGN),
    (dict(dbias=_at(6) + 2, bias_f32=1), _lib.MI_E_ALIGN),
    (dict(dlhs=_at(1)), _lib.MI_E_ARGS),
    (dict(drhs=_at(4)), _lib.MI_E_ARGS),
    (dict(dbias=_at(0)), _lib.MI_E_ARGS),
    (dict(drhs=_at(9)), _lib.MI_E_ARGS),  # the workspace
])
@pytest.mark.parametrize("transposed", [0, 1])
def test_matmul_epilogue_backward(kw, code, transposed):
    fn = _lib.lib().mi_matmul_epilogue_backward_bf16
    assert _code(fn, _mm_bwd(rhs_transposed=transposed, **kw), _at(9), 32 * GIB, None) == code


def _ns(**kw):
    a = dict(grad=_at(0), out=_at(1), batch=2, m=64, n=96, steps=5, dtype=_lib.MI_DTYPE_BF16, a=3.4, b=-4.8, c=2.0, eps=1e-7)
    return _lib.NewtonSchulzArgs(**(a | kw))


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), _lib.MI_E_ARGS),
    (dict(m=-1), _lib.MI_E_ARGS),
    (dict(steps=-1), _lib.MI_E_ARGS),
    (dict(dtype=_lib.MI_DTYPE_F16), _lib.MI_E_ARGS),
    (dict(eps=-1.0), _lib.MI_E_ARGS),
    (dict(eps=float("nan")), _lib.MI_E_ARGS),
    (dict(batch=65536), _lib.MI_E_RANGE),
    (dict(m=40000, n=40000), _lib.MI_E_RANGE),
    (dict(m=1, n=(1 << 20) + 1), _lib.MI_E_RANGE),
    (dict(m=BIG, n=BIG), _lib.MI_E_RANGE),
    (dict(grad=None), _lib.MI_E_ARGS),
    (dict(out=None), _lib.MI_E_ARGS),
    (dict(grad=_at(0) + 2, dtype=_lib.MI_DTYPE_F32), _lib.MI_E_ALIGN),
    (dict(out=_at(0)), _lib.MI_E_ARGS),
    (dict(out=_at(9)), _lib.MI_E_ARGS),
    (dict(grad=_at(9)), _lib.MI_E_ARGS),
    (dict(batch=0, grad=None, out=None), _lib.MI_OK),
    (dict(n=0, grad=None, out=None), _lib.MI_OK),
])
def test_newton_schulz(kw, code):
    assert _code(_lib.lib().mi_newton_schulz, _ns(**kw), _at(9), 32 * GIB, None) == code


def test_newton_schulz_workspace():
    L, need = _lib.lib(), ctypes.c_ulonglong()
    assert _code(L.mi_newton_schulz_workspace, _ns(), ctypes.byref(need)) == 0 and need.value > 0
    assert _code(L.mi_newton_schulz, _ns(), _at(9), need.value - 1, None) == _lib.MI_E_ARGS
    assert _code(L.mi_newton_schulz, _ns(), None, 0, None) == _lib.MI_E_ARGS
    assert L.mi_newton_schulz(None, None, 0, None) == _lib.MI_E_ARGS


def test_configs_are_listed_and_chosen_among():
    cfgs = kl.epilogue_configs()
    assert len(cfgs) == len(set(cfgs)) > 0
    L, c = _lib.lib(), _lib.MiTileCfg()
    assert L.mi_epilogue_config(len(cfgs), ctypes.byref(c)) == _lib.MI_E_ARGS
    assert L.mi_epilogue_config(-1, ctypes.byref(c)) == _lib.MI_E_ARGS
    assert L.mi_epilogue_config(0, None) == _lib.MI_E_ARGS
    need = ctypes.c_ulonglong()
    for M in (1, 16, 33, 128, 1000, 4096, 65536):
        for N in (8, 100, 1024, 8192, 28672):
            for K in (1, 64, 777, 4096, 14336):
                for transposed in (0, 1):
                    if max(M, N) * K >= 2**31 - 2**27:
                        continue
                    assert L.mi_epilogue_default_config(M, N, K, transposed, ctypes.byref(c)) == 0
                    t = kl.TileConfig.from_c(c)
                    assert kl.TileConfig(*(getattr(t, f) for f in ("block_m", "block_n", "block_k", "waves", "lds_stages")),
                                         1, 8, t.variant) in cfgs
                    args = _mm(M=M, N=N, K=K, rhs_transposed=transposed)
                    assert L.mi_matmul_epilogue_workspace(ctypes.byref(args), ctypes.byref(c), ctypes.byref(need)) == 0


def test_python_refuses_what_is_not_on_a_device():
    t = torch.zeros(8, 8, dtype=torch.bfloat16)
    for call in (lambda: kl.layer_norm(t), lambda: kl.layer_norm_backward(t, t, t[:, 0], t[:, 0]),
                 lambda: kl.matmul_epilogue(t, t), lambda: kl.matmul_epilogue_backward(t, t, t),
                 lambda: kl.newton_schulz(t)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    for call in (lambda: kl.layer_norm(None), lambda: kl.matmul_epilogue([1.0], t), lambda: kl.newton_schulz(3)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="activation"):
        kl.matmul_epilogue(t, t, activation="tanh")
    with pytest.raises(ValueError, match="coefficients"):
        kl.newton_schulz(t, coefficients=(1.0, 2.0))
