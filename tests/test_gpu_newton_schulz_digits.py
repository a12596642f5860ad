"""newton_schulz keeps the 16 bits of its iterates in every product, not only those that one rounding leaves visible."""

import pytest

from ns_digits import allowed, distance
from test_gpu_newton_schulz import SHAPES, _grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n", [s for s in SHAPES if min(s) > 30] + [(2048, 2304), (1111, 2500), (2001, 777), (4100, 4100)])
def test_shapes(gpu, m, n, dtype):
    """Each block of the products, X X^T whole and in parts."""
    import kernel_library as kl

    grad = _grad((m, n), dtype, gpu)
    d, most = distance(kl.newton_schulz(grad), grad), allowed(grad)
    print(f"newton_schulz {m}x{n} {dtype}: {d:.2e} of {most:.2e}", flush=True)
    assert d <= most


@pytest.mark.parametrize("shape", [(5, 130, 64), (2, 512, 256), (4, 256, 512), (3, 300, 2000)])
def test_batches(gpu, shape):
    import kernel_library as kl

    grad = _grad(shape, "bfloat16", gpu)
    out = kl.newton_schulz(grad)
    for k in range(shape[0]):
        d, most = distance(out[k], grad[k]), allowed(grad[k])
        print(f"newton_schulz {shape} {k}: {d:.2e} of {most:.2e}", flush=True)
        assert d <= most


@pytest.mark.parametrize("steps", [1, 3, 6])
def test_steps(gpu, steps):
    import kernel_library as kl

    for m, n in ((70, 100), (192, 64), (100, 2100)):
        grad = _grad((m, n), "float32", gpu)
        d, most = distance(kl.newton_schulz(grad, steps=steps), grad, steps), allowed(grad, steps)
        print(f"newton_schulz {m}x{n}, {steps} steps: {d:.2e} of {most:.2e}", flush=True)
        assert d <= most


def test_norms_whose_reciprocal_leaves_fp32(gpu):
    """fp32 gradients near either end of its range, without an eps: 1 / norm is past the largest number, or has lost
    digits under the smallest normal one."""
    import torch

    import kernel_library as kl

    for m, n in ((70, 100), (129, 64)):
        for scale in (1e-41, 3e-43, 5e37):
            grad = _grad((m, n), "float32", gpu, scale=1.0)
            grad = (grad.double() / float(grad.abs().max()) * scale * 5).float()
            assert torch.isfinite(grad).all() and float(grad.abs().max()) > 0
            d, most = distance(kl.newton_schulz(grad, eps=0.0), grad, eps=0.0), allowed(grad * 1.0, eps=0.0)
            print(f"newton_schulz {m}x{n} {scale}: {d:.2e} of {most:.2e}", flush=True)
            assert d <= most
    zero = torch.zeros(40, 50, device=gpu)
    assert (kl.newton_schulz(zero, eps=1e-42) == 0).all()
