"""The check of newton_schulz's digits (ns_digits) sees what it is for: emulations that lose some."""

import pytest
import torch

from ns_digits import LOSSES, allowed, distance, emulated

# Sizes of the kernel's tests, small and long, turned, and ones whose X X^T goes in parts.
SHAPES = [(31, 33), (65, 63), (40, 300), (257, 129), (777, 100), (100, 2100), (512, 1024), (640, 4000)]


def _grad(shape):
    g = torch.Generator().manual_seed(sum(shape))
    m, n = shape
    r = max(1, min(m, n) // 8)
    low = torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g)
    return (1e-3 * (low + torch.randn(m, n, generator=g))).bfloat16()


@pytest.mark.parametrize("shape", SHAPES)
def test_each_loss_is_seen(shape):
    grad = _grad(shape)
    bound = allowed(grad)
    assert bound < 1.1e-3
    for name, loss in LOSSES.items():
        assert distance(emulated(grad, **loss), grad) > 1.25 * bound, name
