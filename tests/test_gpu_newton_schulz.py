"""newton_schulz against its plain 64-bit form."""

import pytest

from block_oracle import half_step
from block_oracle import newton_schulz as ns64

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 9), (9, 1), (2, 3), (31, 33), (64, 64), (65, 63), (40, 300), (300, 40), (128, 513), (200, 200),
          (257, 129), (777, 100), (1, 5000), (512, 1024), (100, 2100), (3001, 129), (640, 4000)]


def _grad(shape, dtype, gpu, seed=0, scale=1e-3):
    import torch

    g = torch.Generator().manual_seed(sum(shape) + seed)
    m, n = shape[-2:]
    r = max(1, min(m, n) // 8)
    low = torch.randn(*shape[:-1], r, generator=g) @ torch.randn(*shape[:-2], r, n, generator=g)
    return (scale * (low + torch.randn(*shape, generator=g))).to(getattr(torch, dtype)).to(gpu)


def _check(out, grad, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """Each matrix's error, in the 2-norm, against the 64-bit form's.

    One rounding of each element to bf16 is at most 2^-8 of the whole.  A step rounds X, A and B to 2^-18 each, leaves
    2^-18 of each product out and sums in fp32; a relative perturbation d of an iterate comes out of a step at most
    (|a| + 3|b| + 5|c|) d with singular values up to 1.3, but in the 2-norm of the whole, whose singular values are
    spread, about the slope at 0, |a|, at worst: 5 steps give 3.45^5 = 488 of the first step's 3 * 2^-18."""
    import torch

    e = ns64(grad, steps, coefficients, eps)
    a = out.double()
    assert a.shape == e.shape and torch.isfinite(a).all()
    norm = torch.linalg.matrix_norm(e)
    err = torch.linalg.matrix_norm(a - e)
    bound = half_step(torch.bfloat16) + 3 * 2.0**-18 * sum(max(1.0, abs(coefficients[0])) ** k for k in range(1, steps + 1))
    assert bool((err <= bound * norm + 1e-30).all()), (err / norm, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(gpu, m, n, dtype):
    import torch

    import kernel_library as kl

    print(f"newton_schulz {m}x{n} {dtype}", flush=True)
    grad = _grad((m, n), dtype, gpu)
    out = kl.newton_schulz(grad)
    assert out.shape == (m, n) and out.dtype == torch.bfloat16
    _check(out, grad)


@pytest.mark.parametrize("shape", [(3, 40, 72), (5, 130, 64), (2, 512, 256), (4, 1, 7), (2, 300, 1000), (3, 300, 2000)])
def test_a_batch_is_its_matrices(gpu, shape):
    import torch

    import kernel_library as kl

    print(f"newton_schulz {shape}", flush=True)
    grad = _grad(shape, "bfloat16", gpu)
    grad[1] *= 100  # a scale of its own
    out = kl.newton_schulz(grad)
    _check(out, grad)
    again = torch.empty_like(out)
    assert kl.newton_schulz(grad, out=again) is again and (again == out).all()
    for k in range(shape[0]):
        _check(kl.newton_schulz(grad[k].contiguous()), grad[k])


@pytest.mark.parametrize("steps", [0, 1, 2, 7])
def test_steps_and_coefficients(gpu, steps):
    import kernel_library as kl

    for m, n in ((70, 100), (128, 64), (64, 192)):
        grad = _grad((m, n), "float32", gpu)
        _check(kl.newton_schulz(grad, steps=steps), grad, steps)
        cubic = (1.5, -0.5, 0.0)
        _check(kl.newton_schulz(grad, steps=steps, coefficients=cubic, eps=0.0), grad, steps, cubic, 0.0)


def test_larger_products(gpu):
    """Sizes that take each block of the products, whole and ragged."""
    import kernel_library as kl

    for m, n in ((2048, 2304), (1111, 2500), (2500, 1111), (4100, 4100)):
        print(f"newton_schulz {m}x{n}", flush=True)
        grad = _grad((m, n), "bfloat16", gpu)
        _check(kl.newton_schulz(grad), grad)


def test_the_result_is_nearly_orthogonal(gpu):
    """Singular values that the iteration takes into its band, on a matrix with a spread of them."""
    import torch

    import kernel_library as kl

    g = torch.Generator().manual_seed(1)
    u, _ = torch.linalg.qr(torch.randn(96, 96, generator=g, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(160, 96, generator=g, dtype=torch.float64))
    grad = (u * torch.logspace(0, -2, 96, dtype=torch.float64)) @ v.T
    s = torch.linalg.svdvals(kl.newton_schulz(grad.float().to(gpu)).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


def test_gradients_out_of_the_ordinary(gpu):
    import torch

    import kernel_library as kl

    zero = torch.zeros(40, 70, device=gpu)
    assert (kl.newton_schulz(zero) == 0).all()
    for scale in (1e-25, 1e-12, 1e15, 1e28):  # squares past fp32's range either way
        grad = _grad((50, 90), "float32", gpu, scale=scale)
        _check(kl.newton_schulz(grad, eps=0.0), grad, eps=0.0)
    rank_one = torch.outer(torch.arange(1, 51, device=gpu).float(), torch.ones(30, device=gpu))
    _check(kl.newton_schulz(rank_one), rank_one)
    bad = _grad((40, 70), "float32", gpu)
    bad[3, 4] = float("nan")
    assert torch.isnan(kl.newton_schulz(bad)).all()
    two = torch.stack([_grad((40, 70), "float32", gpu), bad])
    out = kl.newton_schulz(two)
    assert torch.isnan(out[1]).all()
    _check(out[0], two[0])
    assert kl.newton_schulz(torch.empty(0, 5, 6, device=gpu)).shape == (0, 5, 6)
    assert kl.newton_schulz(torch.empty(0, 6, device=gpu)).shape == (0, 6)


def test_only_the_output_is_written(gpu):
    import torch

    import kernel_library as kl

    for m, n, off in ((33, 65, 0), (33, 65, 1), (64, 128, 8), (128, 64, 3)):
        grad = _grad((m, n), "bfloat16", gpu)
        big = torch.full((m * n + 1024,), 7.0, dtype=torch.bfloat16, device=gpu)
        out = big[512 + off:512 + off + m * n].view(m, n)
        kl.newton_schulz(grad, out=out)
        _check(out, grad)
        assert (big[:512 + off] == 7).all() and (big[512 + off + m * n:] == 7).all()


@pytest.mark.parametrize("shape", [(2, 130, 200), (2, 100, 3000)])
def test_same_bits_on_streams_and_in_graphs(gpu, shape):
    import torch

    import kernel_library as kl

    grad = _grad(shape, "float32", gpu)
    want = kl.newton_schulz(grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kl.newton_schulz(grad)
    torch.cuda.synchronize()
    assert (want == other).all()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kl.newton_schulz(grad)
        graphs.append((graph, out))
    for k in range(3):
        grad.copy_(_grad(shape, "float32", gpu, seed=k + 1))
        want = kl.newton_schulz(grad)
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert (want == out).all()
