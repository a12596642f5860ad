"""The tile configs that matmul_epilogue compiles: what a caller may pass, and what the library chooses."""

import dataclasses

import pytest

from test_gpu_matmul_epilogue import _check, _check_backward, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group_m", [2**31 - 1, 2**30, 2**29 + 1, 3, 0])
@pytest.mark.parametrize("transposed", [False, True])
def test_raster_groups_of_any_size(gpu, transposed, group_m):
    """A group of more tile rows than there are is one of all of them: the same result, in parts too."""
    import torch

    import kernel_library as kl
    from kernel_library import TileConfig

    # Four and two columns of tiles: 4 * 2^30 is 0 in 32 bits, 2 * (2^31 - 1) negative.
    for M, N, K in ((300, 500, 264), (130, 136, 1000)):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
        for cfg in (TileConfig(128, 128, 64, 4, 4), TileConfig(64, 64, 64, 4, 2)):
            for parts in (1, 2):
                c = dataclasses.replace(cfg, split_k=parts, group_m=group_m)
                print(f"{c.name} {M}x{N}x{K} {transposed}", flush=True)
                out = kl.matmul_epilogue(lhs, rhs, b, "gelu", r, rhs_transposed=transposed, cfg=c)
                want = kl.matmul_epilogue(lhs, rhs, b, "gelu", r, rhs_transposed=transposed,
                                          cfg=dataclasses.replace(c, group_m=8))
                assert torch.equal(out, want)
                _check(lhs, rhs, b, "gelu", r, transposed, out)


@pytest.mark.parametrize("transposed", [False, True])
def test_every_compiled_config(gpu, transposed):
    """Each that the library lists, at ragged sizes, whole and split."""
    import torch

    import kernel_library as kl

    ran = 0
    for cfg in kl.epilogue_configs():
        for M, N, K in ((70, 520, 456), (389, 267, 1000), (17, 1032, 203)):
            lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed, "float32")
            pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
            for parts in (1, 2, 4):
                c = dataclasses.replace(cfg, split_k=parts)
                print(f"{c.name} {M}x{N}x{K} {transposed}", flush=True)
                out = kl.matmul_epilogue(lhs, rhs, b, "silu", r, rhs_transposed=transposed, pre=pre, cfg=c)
                _check(lhs, rhs, b, "silu", r, transposed, out, pre)
                ran += 1
    assert ran == 9 * len(kl.epilogue_configs())


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("M,N,K", [(16, 28672, 8192), (16, 8192, 28672), (1, 8192, 16392), (70, 16392, 8200)])
def test_weights_past_the_last_level_cache(gpu, M, N, K, transposed):
    """More than 256 MiB of rhs: what the library chooses there, and the gradients."""
    import ctypes

    import torch

    import kernel_library as kl
    from kernel_library import _lib

    c = _lib.MiTileCfg()
    assert _lib.lib().mi_epilogue_default_config(M, N, K, int(transposed), ctypes.byref(c)) == 0
    assert c.variant == 1 or M > 64, "few rows read such a rhs non-temporally"
    print(f"{M}x{N}x{K} {transposed}: {kl.TileConfig.from_c(c).name}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(M + N)
    lhs, r = (torch.randn(*s, generator=g, device=gpu).bfloat16() for s in ((M, K), (M, N)))
    rhs = (torch.randn(*((N, K) if transposed else (K, N)), generator=g, device=gpu) / K**0.5).bfloat16()
    b = torch.randn(N, generator=g, device=gpu)
    pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
    out = kl.matmul_epilogue(lhs, rhs, b, "silu", r, rhs_transposed=transposed, pre=pre)
    _check(lhs, rhs, b, "silu", r, transposed, out, pre)
    _check_backward(r, lhs, rhs, "silu", pre, transposed,
                    *kl.matmul_epilogue_backward(r, lhs, rhs, "silu", pre, b, rhs_transposed=transposed))
