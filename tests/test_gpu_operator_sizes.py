"""The operators at the ends of the sizes that their documentation allows."""

import pytest

from block_oracle import half_step, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [2**26 + 65, 2**28 - 63, 2**28])
def test_parameter_gradients_of_the_longest_rows(gpu, D):
    """A launch holds under 2^32 threads; a block of 1024 for each 64 columns of 2^28 would be as many.

    One row, so that each sum has one term: dbias is dout itself, dweight dout * (x - mean) * rstd with a difference
    rounded once, two products, and one rounding to bf16."""
    import torch

    import kernel_library as kl

    print(f"layer_norm_backward 1x{D}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(D)
    x, dout, w = (torch.randn(1, D, generator=g, device=gpu, dtype=torch.bfloat16) for _ in range(3))
    mean, rstd = torch.full((1,), 0.25, device=gpu), torch.full((1,), 2.0, device=gpu)
    dx, dw, db = kl.layer_norm_backward(dout, x, mean, rstd, w[0], w[0], need_dx=False)
    assert dx is None and torch.equal(db, dout[0])
    step = 1 << 26
    for at in range(0, D, step):
        xs, ds = x[0, at:at + step].double(), dout[0, at:at + step].double()
        e = ds * (xs - 0.25) * 2.0
        within(dw[at:at + step], e, half_step(torch.bfloat16) * e.abs() * (1 + 2.0**-20) + 2.0**-22 * ds.abs() * (xs.abs() + 0.25))


def test_bias_gradients_of_the_widest_outputs(gpu):
    import torch

    import kernel_library as kl

    for N in (2**28 - 63, 2**28):
        print(f"matmul_epilogue_backward 1x{N}x0", flush=True)
        g = torch.Generator(device=gpu).manual_seed(N)
        dout = torch.randn(1, N, generator=g, device=gpu, dtype=torch.bfloat16)
        lhs, rhs = torch.empty(1, 0, dtype=torch.bfloat16, device=gpu), torch.empty(0, N, dtype=torch.bfloat16, device=gpu)
        dlhs, drhs, db = kl.matmul_epilogue_backward(dout, lhs, rhs, bias=torch.empty(N, device=gpu))
        assert dlhs.shape == (1, 0) and drhs.shape == (0, N) and torch.equal(db, dout[0].float())
