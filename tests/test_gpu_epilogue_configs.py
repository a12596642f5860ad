"""The tile configs that matmul_epilogue compiles: what a caller may pass, and what the library chooses."""

import dataclasses

import pytest

from test_gpu_matmul_epilogue import _check, _inputs

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
