"""matmul_fp8 where the products of two scales leave fp32's normal range."""

import pytest

from block_oracle import half_step, within
from step_oracle import matmul_fp8 as mm64
from step_oracle import spread
from test_gpu_fp8 import _check_product

pytestmark = pytest.mark.gpu


def _operands(M, N, K, scales, square, exponents, gpu):
    """Positive values from 224 to 448, whose sums over a block are 2^22.6 at least, and scales of these exponents."""
    import torch

    g = torch.Generator().manual_seed(M + N + K)
    kb = -(-K // 128)

    def values(rows):
        return (224 + 224 * torch.rand(rows, K, generator=g)).to(torch.float8_e4m3fn).to(gpu)

    def some(rows, exponent):
        if scales == "e8m0":
            return torch.randint(127 + exponent, 130 + exponent, (rows, kb), generator=g,
                                 dtype=torch.uint8).view(torch.float8_e8m0fnu).to(gpu)
        return torch.ldexp(1 + torch.rand(rows, kb, generator=g), torch.tensor(exponent)).to(gpu)

    return values(M), some(M, exponents[0]), values(N), some(-(-N // 128) if square else N, exponents[1])


@pytest.mark.parametrize("scales,square", [("float32", True), ("float32", False), ("e8m0", False)])
@pytest.mark.parametrize("exponents", [(-63, -63), (-100, -26), (-26, -100), (-74, -74), (-100, -48), (-48, -100)])
def test_small_scales(gpu, exponents, scales, square):
    """Products of scales down to 2^-126 are as exact as any.  Below, fp32 ones are rounded to multiples of 2^-149, so
    each block's values' products are off by at most 2^-150 of their unscaled sum; powers of two are not.  Results are
    2^-126 at least: normal numbers."""
    import torch

    import kernel_library as kl

    M, N, K = 140, 200, 500
    a = _operands(M, N, K, scales, square, exponents, gpu)
    low = sum(exponents) < -126
    for cfg in (None, *kl.fp8_configs()):
        print(f"matmul_fp8 {scales} {square} 2^{exponents} {cfg}", flush=True)
        out = kl.matmul_fp8(*a, cfg=cfg)
        if not low or scales == "e8m0":
            _check_product(out, *a)
            continue
        lhs, ls, rhs, rs = a
        e, mag = mm64(*a)
        assert float(e.min()) >= 2.0**-126
        unscaled = lhs.double() @ rhs.double().t().contiguous()
        exact = 7 * 2.0**-13 * mag + (K / 8 + 4 * (K // 128 + 1) + 20) * 2.0**-23 * mag + half_step(out.dtype) * e
        within(out, e, exact + 2.0**-150 * unscaled * (1 + half_step(out.dtype)))
        # What comes of the products as fp32 has them, to the tolerance of any other product.
        s = spread(ls, False, M, K)[:, ::128][:, None] * spread(rs, square, N, K)[:, ::128][None]
        blocks = torch.stack([lhs[:, k:k + 128].double() @ rhs[:, k:k + 128].double().t().contiguous() for k in range(0, K, 128)], -1)
        within(out, (blocks * s.float().double()).sum(-1), exact)
