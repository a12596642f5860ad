"""The raster group of a config: past the tile rows there are, it is one group of all of them."""

import dataclasses

import pytest

pytestmark = pytest.mark.gpu

M, N, K = 264, 520, 512  # whole and partial tiles of every block


def _operands(func, gpu):
    import torch

    g = torch.Generator().manual_seed(7)
    f32 = func == "matmul_lhsT_rhs_f32"
    t = torch.float32 if f32 else torch.bfloat16
    lhs_shape = (K, M) if func.startswith("matmul_lhsT") else (M, K)
    return [torch.randn(*s, generator=g).to(t).to(gpu) for s in (lhs_shape, (K, N))]


@pytest.mark.parametrize("func", ["matmul_lhsT_rhs", "matmul_lhsT_rhs_f32", "matmul_lhs_rhs", "rmsnorm_matmul"])
def test_groups_past_the_tile_rows(gpu, func):
    """Products by the tile columns, 2^30 and 2^31 - 1 wrap in 32 bits: every compiled config, against group_m 8."""
    import torch

    import kernel_library as kl

    lhs, rhs = _operands(func, gpu)
    call = getattr(kl, func.removesuffix("_f32"))
    ran = 0
    for cfg in kl.compiled_configs(func):
        if kl.check(func, cfg, M, N, K)[0]:
            continue
        print(f"{func} {cfg.name}", flush=True)
        want = call(lhs, rhs, cfg=dataclasses.replace(cfg, group_m=8))
        for group in (2**31 - 1, 2**30):
            assert torch.equal(call(lhs, rhs, cfg=dataclasses.replace(cfg, group_m=group)), want), (cfg.name, group)
        ran += 1
    assert ran
