"""quantize_fp8 where scales are small and quotients lie next to the border between two 8-bit values."""

import pytest

from step_oracle import LIMIT
from step_oracle import quantize as q64
from test_gpu_fp8 import _same_values, _t

pytestmark = pytest.mark.gpu


def near_borders(dtype, rows, lowest, highest, seed):
    """[rows, 128] fp32: row r's scale has an exponent in [lowest, highest) and any significand, every other row's one
    within 64 steps of a power of two; its values are that scale's products with the borders between neighbours among
    the type's smallest values, and the fp32 values beside those, which a quotient that is off in its last place takes
    for their neighbours."""
    import torch

    g = torch.Generator().manual_seed(seed)
    limit = LIMIT[dtype]
    part = torch.randint(1 << 23, (rows, 1), generator=g)
    part[::2] = torch.randint(-64, 64, (rows // 2, 1), generator=g) % (1 << 23)
    scale = torch.ldexp(1 + part.double() / (1 << 23), torch.randint(lowest, highest, (rows, 1), generator=g))
    most = (limit * scale).float()
    scale = (most.double() / limit).float().double()
    every = torch.arange(256, dtype=torch.uint8).view(dtype).double()
    every = torch.unique(every[torch.isfinite(every)])
    border = ((every[1:] + every[:-1]) / 2)[every[1:] > 0][:10]
    x = (scale * border[torch.randint(len(border), (rows, 128), generator=g)]).float()
    bits = x.view(torch.int32) + torch.randint(-1, 2, (rows, 128), generator=g, dtype=torch.int32)
    x = bits.view(torch.float32) * (1 - 2 * torch.randint(2, (rows, 128), generator=g))
    x[:, :1] = most
    return x


@pytest.mark.parametrize("dtype", ["e4m3", "e5m2"])
@pytest.mark.parametrize("lowest,highest", [(-100, -96), (-96, -90), (-90, -78), (-78, -40), (-12, 12)])
def test_small_scales(gpu, dtype, lowest, highest):
    """Residuals of the quotient that are below fp32's normal range: values are the definition's all the same."""
    import torch

    import kernel_library as kl

    x = near_borders(_t(dtype), 1 << 15, lowest, highest, -lowest).to(gpu)
    eq, es = q64(x, False, _t(dtype))
    q, s, *_ = kl.quantize_fp8(x, dtype=_t(dtype), transposed=True)
    _same_values(s, es)
    _same_values(q, eq)
    _, _, q, s = kl.quantize_fp8(x.t().contiguous(), dtype=_t(dtype), transposed=True)
    _same_values(s, es)
    _same_values(q, eq)
    # One scale for 128 x 128 values: those of a row whose scale is the largest of all.
    y = x[:256].repeat_interleave(128, 0)
    q, s, q_t, s_t = kl.quantize_fp8(y, (128, 128), dtype=_t(dtype), transposed=True)
    _same_values(s, es[:256])
    _same_values(q, eq[:256].repeat_interleave(128, 0))
    _same_values(q_t, eq[:256].repeat_interleave(128, 0).t())
    _same_values(s_t, es[:256].t())
    # Rows of zeros beside such, and as bf16 (which has few of the borders).
    z = x[:384].clone()
    z[::3] = 0.0
    for v in (z, z.bfloat16()):
        for w in (v, v.t().contiguous()):
            q, s, q_t, s_t = kl.quantize_fp8(w, dtype=_t(dtype), transposed=True)
            for a, b, u in ((q, s, w), (q_t, s_t, w.t())):
                eq2, es2 = q64(u, False, _t(dtype))
                _same_values(b, es2)
                _same_values(a, eq2)
    assert torch.isfinite(s).all()
