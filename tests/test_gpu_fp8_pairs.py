"""matmul_fp8_backward: both products in one launch, and each by itself."""

import ctypes

import pytest

from test_gpu_fp8 import _rows, _t
from test_gpu_step import _step_operands

pytestmark = pytest.mark.gpu


def _launches(call):
    """Kernels that ``call`` launches: the nodes of its graph, of the runtime that torch has loaded."""
    import torch

    with open("/proc/self/maps") as f:
        paths = {line.split()[-1] for line in f if "libamdhip64" in line}
    assert len(paths) == 1, paths
    nodes = ctypes.CDLL(paths.pop()).hipGraphGetNodes
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    count = ctypes.c_size_t()
    assert nodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    return count.value


SHAPES = [(1, 1, 1), (5, 3, 200), (64, 64, 64), (130, 700, 500), (1000, 520, 777), (300, 2000, 136), (256, 256, 256),
          (40, 4000, 2000), (2048, 4096, 2048)]


@pytest.mark.parametrize("scales,square", [("float32", False), ("float32", True), ("e8m0", False)])
def test_a_pair_gives_what_each_gives(gpu, scales, square):
    """Bit by bit: a product's values depend on its blocks only where K is split into parts, which a pair's is not, and
    which adds a launch to a product by itself."""
    import torch

    import kernel_library as kl

    paired = apart = 0
    for M, N, K in SHAPES:
        _, _, a, b = _step_operands(gpu, M, N, K, scales, square)
        dout = _rows(M, N, 3, gpu).bfloat16()
        for dt in ("e4m3", "e5m2"):
            calls = [lambda kw=kw: kl.matmul_fp8_backward(dout, *a[2:], *b[2:], dtype=_t(dt), **kw)
                     for kw in ({}, dict(need_drhs=False), dict(need_dlhs=False))]
            (dl, dr), (dl1, none), (none2, dr1) = (c() for c in calls)
            assert none is None and none2 is None
            n, left, right = (_launches(c) for c in calls)
            print(f"matmul_fp8_backward {M}x{N}x{K} {scales} {square} {dt}: {n} launches, alone {left} and {right}", flush=True)
            if n == 2:  # the gradient's 8-bit form (with padded copies, if any), and both products
                paired += 1
                if left == 2:  # the same, and one product: not split
                    assert torch.equal(dl, dl1), (M, N, K, dt)
                if right == 2:
                    assert torch.equal(dr, dr1), (M, N, K, dt)
            else:
                apart += 1
                assert torch.equal(dl, dl1) and torch.equal(dr, dr1), (M, N, K, dt)
    assert paired > 0 and apart > 0, (paired, apart)
