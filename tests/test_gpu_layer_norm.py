"""layer_norm and its gradients against their plain 64-bit forms."""

import pytest

from block_oracle import half_step, within
from block_oracle import layer_norm as ln64
from block_oracle import layer_norm_backward as ln_bwd64

pytestmark = pytest.mark.gpu

# A row per wave, a few waves per row, rows longer than registers hold; whole vectors and odd sizes.
SIZES = [(1, 1), (1, 8), (3, 7), (300, 17), (700, 32), (257, 33), (5, 64), (9, 100), (4, 512), (33, 513), (2, 1024), (7, 1501), (17, 2048), (5, 2056),
         (3, 4096), (300, 777), (1, 4104), (2, 8192), (3, 8191), (2, 16384), (2, 16392), (1, 16383), (2, 32768), (1, 40001)]
TYPES = [("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16"), ("float32", "float32")]


def _inputs(rows, D, dtype, wt, gpu, seed=0):
    import torch

    g = torch.Generator().manual_seed(1000 * rows + D + seed)
    x = torch.randn(rows, D, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + torch.randn(rows, 1, generator=g)
    w, b = 1 + 0.1 * torch.randn(D, generator=g), 0.1 * torch.randn(D, generator=g)
    dout = torch.randn(rows, D, generator=g)
    t = getattr(torch, dtype)
    return x.to(t).to(gpu), w.to(getattr(torch, wt)).to(gpu), b.to(getattr(torch, wt)).to(gpu), dout.to(t).to(gpu)


def _check_forward(x, w, b, eps, y, mean, rstd):
    """The statistics and y, each within what fp32 sums and one rounding may lose.

    A lane sums at most 64 values and a row at most 10 levels of pairs and 16 waves (rows past registers: D / 1024 in
    line), so a sum is off by n 2^-24 of its terms' magnitudes, n = 90 + D / 1024; the second pass takes the mean's
    error out again (mean off by n 2^-24 of the centred magnitudes, and one rounding of its own size)."""
    import torch

    D = x.shape[-1]
    n = (90 + D / 1024) * 2.0**-24
    ey, em, er = ln64(x, w, b, eps)
    c = (x.double() - em[..., None]).abs()
    mean_tol = n * c.mean(-1) + n * n * x.double().abs().mean(-1) + 2.0**-23 * em.abs()
    within(mean, em, mean_tol)
    within(rstd, er, er * 4 * n + 1e-30)
    scale = er[..., None] * (w.double().abs() if w is not None else 1.0)
    inner = scale * (c * 6 * n + mean_tol[..., None]) + 2.0**-23 * (b.double().abs() if b is not None else 0.0)
    inner = inner + 2.0**-22 * ey.abs()
    within(y, ey, inner + (half_step(x.dtype) if x.dtype != torch.float32 else 0.0) * ey.abs() + 1e-7 * (x.dtype == torch.float16))


def _check_backward(dout, x, mean, rstd, w, dx, dw, db):
    import torch

    D, rows = x.shape[-1], max(1, x.numel() // x.shape[-1])
    edx, edw, edb = ln_bwd64(dout, x, mean, rstd, w)
    n = (90 + D / 1024) * 2.0**-24
    xh = ((x.double() - mean.double()[..., None]) * rstd.double()[..., None]).abs()
    # x - mean is rounded once, relative to the larger of the two.
    dxh = (x.double().abs() + mean.double().abs()[..., None]) * rstd.double()[..., None] * 2.0**-23 + xh * 2.0**-23
    dy = dout.double().abs()
    g = dy * (w.double().abs() if w is not None else 1.0)
    mg, mgx, mgd = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True), (g * dxh).mean(-1, keepdim=True)
    inner = rstd.double()[..., None] * ((n + 2.0**-22) * (g + mg + xh * mgx) + dxh * mgx + xh * mgd)
    within(dx, edx, inner + half_step(x.dtype) * edx.abs() + 1e-7 * (x.dtype == torch.float16))
    # A column's sum: at most rows terms in line (fewer by far: blocks, waves and parts are added by levels).
    m = (min(rows, 600) + 40) * 2.0**-24
    for a, e, mag in ((dw, edw, (dy * xh).reshape(-1, D).sum(0)), (db, edb, dy.reshape(-1, D).sum(0))):
        extra = (dy * dxh).reshape(-1, D).sum(0) if a is dw else 0.0
        if a is not None:
            within(a, e, m * mag + extra + half_step(a.dtype) * e.abs() + 1e-6 * (a.dtype == torch.float16))


@pytest.mark.parametrize("dtype,wt", TYPES)
@pytest.mark.parametrize("rows,D", SIZES)
def test_forward_and_gradients(gpu, rows, D, dtype, wt):
    import kernel_library as kl

    print(f"layer_norm {rows}x{D} {dtype} {wt}", flush=True)
    x, w, b, dout = _inputs(rows, D, dtype, wt, gpu)
    y, mean, rstd = kl.layer_norm(x, w, b, eps=1e-5, stats=True)
    assert y.dtype == x.dtype and y.shape == x.shape and mean.shape == rstd.shape == (rows,)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    dx, dw, db = kl.layer_norm_backward(dout, x, mean, rstd, w, b)
    assert dx.dtype == x.dtype and dw.dtype == db.dtype == w.dtype
    _check_backward(dout, x, mean, rstd, w, dx, dw, db)


@pytest.mark.parametrize("rows", [1, 2, 255, 2049, 5000])
@pytest.mark.parametrize("D", [96, 1501, 4096, 16400])
def test_many_rows(gpu, rows, D):
    """Row counts around the blocks of the gradient's column sums."""
    import kernel_library as kl

    if rows * D > 9_000_000:
        pytest.skip("longer than this check needs")
    print(f"layer_norm rows {rows}x{D}", flush=True)
    x, w, b, dout = _inputs(rows, D, "bfloat16", "float32", gpu)
    y, mean, rstd = kl.layer_norm(x, w, b, stats=True)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    _check_backward(dout, x, mean, rstd, w, *kl.layer_norm_backward(dout, x, mean, rstd, w, b))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("D", [64, 1501, 4096])
def test_parts_that_are_not_there(gpu, D, dtype):
    import kernel_library as kl

    x, w, b, dout = _inputs(11, D, dtype, dtype, gpu)
    y, mean, rstd = kl.layer_norm(x, stats=True)
    _check_forward(x, None, None, 1e-5, y, mean, rstd)
    assert (kl.layer_norm(x) == y).all()
    dx, dw, db = kl.layer_norm_backward(dout, x, mean, rstd)
    assert dw is None and db is None
    _check_backward(dout, x, mean, rstd, None, dx, None, None)
    # One parameter at a time, and the column sums alone.
    y1, m1, r1 = kl.layer_norm(x, w, stats=True)
    _check_forward(x, w, None, 1e-5, y1, m1, r1)
    full = kl.layer_norm_backward(dout, x, mean, rstd, w, b)
    for args, keep in (((w, None), (0, 1)), ((None, b), (2,))):
        got = kl.layer_norm_backward(dout, x, mean, rstd, *args)
        for k in keep:
            assert (got[k] == full[k]).all()
    none, dw, db = kl.layer_norm_backward(dout, x, mean, rstd, w, b, need_dx=False)
    assert none is None and (dw == full[1]).all() and (db == full[2]).all()


def test_strided_and_broadcast_rows(gpu):
    import torch

    import kernel_library as kl

    for D, ld in ((64, 200), (64, 72), (1501, 1600), (4096, 5000)):
        x, w, b, dout = _inputs(9, D, "bfloat16", "bfloat16", gpu)
        wide = torch.full((9, ld), float("nan"), dtype=x.dtype, device=gpu)
        wide_d = wide.clone()
        wide[:, 3:3 + D] = x
        wide_d[:, 5:5 + D] = dout
        y, mean, rstd = kl.layer_norm(x, w, b, stats=True)
        ys, ms, rs = kl.layer_norm(wide[:, 3:3 + D], w, b, stats=True)
        # (Other loads, so another order of the sums: close, not equal.)
        _check_forward(x, w, b, 1e-5, ys, ms, rs)
        got = kl.layer_norm_backward(wide_d[:, 5:5 + D], wide[:, 3:3 + D], mean, rstd, w, b)
        _check_backward(dout, x, mean, rstd, w, *got)
        # One row for all: its gradient has a row for each.
        row = x[:1].expand(9, D)
        ye, me, re = kl.layer_norm(row, w, b, stats=True)
        _check_forward(row, w, b, 1e-5, ye, me, re)
        _check_backward(dout[:1].expand(9, D), row, me, re, w, *kl.layer_norm_backward(dout[:1].expand(9, D), row, me, re, w, b))


def test_leading_dimensions_and_out(gpu):
    import torch

    import kernel_library as kl

    x, w, b, dout = _inputs(24, 96, "float16", "float16", gpu)
    y, mean, rstd = kl.layer_norm(x, w, b, stats=True)
    y3, m3, r3 = kl.layer_norm(x.view(2, 3, 4, 96), w, b, stats=True)
    assert y3.shape == (2, 3, 4, 96) and m3.shape == (2, 3, 4)
    assert (y3.view(24, 96) == y).all() and (m3.view(24) == mean).all() and (r3.view(24) == rstd).all()
    dx3, dw3, db3 = kl.layer_norm_backward(dout.view(2, 3, 4, 96), x.view(2, 3, 4, 96), m3, r3, w, b)
    dx, dw, db = kl.layer_norm_backward(dout, x, mean, rstd, w, b)
    assert (dx3.view(24, 96) == dx).all() and (dw3 == dw).all() and (db3 == db).all()
    one = kl.layer_norm(x[0], w, b)
    assert one.shape == (96,) and (one == y[0]).all()
    around = torch.full((26, 96), 7.0, dtype=x.dtype, device=gpu)
    got = kl.layer_norm(x, w, b, out=around[1:25])
    assert got.data_ptr() == around[1:25].data_ptr() and (got == y).all()
    assert (around[0] == 7).all() and (around[25] == 7).all()
    # Rows that start off 16 bytes.
    flat = torch.zeros(24 * 96 + 1, dtype=x.dtype, device=gpu)
    off = flat[1:].view(24, 96)
    off.copy_(x)
    _check_forward(x, w, b, 1e-5, *kl.layer_norm(off, w, b, stats=True))


def test_no_rows(gpu):
    import torch

    import kernel_library as kl

    w = torch.ones(40, device=gpu)
    x = torch.empty(0, 40, device=gpu)
    y, mean, rstd = kl.layer_norm(x, w, w, stats=True)
    assert y.shape == (0, 40) and mean.shape == (0,)
    for dtype in (torch.float32,):
        dx, dw, db = kl.layer_norm_backward(x, x, mean, rstd, w, w)
        assert dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all() and dw.dtype == dtype


@pytest.mark.parametrize("D", [64, 777, 4096, 20000])
def test_rows_that_are_constant_or_far_or_not_finite(gpu, D):
    import torch

    import kernel_library as kl

    x = torch.randn(8, D, generator=torch.Generator().manual_seed(D)).to(gpu)
    x[1] = 3.0                      # no variance: y is the bias
    x[2] += 4096.0                  # far from 0 against its spread
    x[3, D // 2] = float("inf")
    x[4, 0] = float("nan")
    x[5] *= 1e18                    # a variance near the largest number
    x[6] *= 1e-20                   # a variance under eps
    w, b = torch.full((D,), 0.5, device=gpu), torch.full((D,), 0.25, device=gpu)
    y, mean, rstd = kl.layer_norm(x, w, b, stats=True)
    assert (y[1] == 0.25).all() and float(mean[1]) == 3.0
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all() and torch.isnan(rstd[3]) and torch.isnan(rstd[4])
    good = [0, 2, 5, 6, 7]
    _check_forward(x[good], w, b, 1e-5, y[good], mean[good], rstd[good])


def test_same_bits_every_time_and_under_a_graph(gpu):
    import torch

    import kernel_library as kl

    x, w, b, dout = _inputs(700, 1504, "bfloat16", "float32", gpu)
    mean, rstd = kl.layer_norm(x, w, b, stats=True)[1:]
    first = kl.layer_norm_backward(dout, x, mean, rstd, w, b)
    for _ in range(3):
        assert all((p == q).all() for p, q in zip(first, kl.layer_norm_backward(dout, x, mean, rstd, w, b)))
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, m, r = kl.layer_norm(x, w, b, stats=True)
            outs.append((y, *kl.layer_norm_backward(dout, x, m, r, w, b)))
        graphs.append(graph)
    for step in range(3):
        x.copy_(_inputs(700, 1504, "bfloat16", "float32", gpu, seed=step)[0])
        y, m, r = kl.layer_norm(x, w, b, stats=True)
        eager = (y, *kl.layer_norm_backward(dout, x, m, r, w, b))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in outs:
            assert all((p == q).all() for p, q in zip(eager, got))


def test_gradient_against_differences(gpu):
    """The directional derivative of the 64-bit forward form, by central differences."""
    import torch

    import kernel_library as kl

    x, w, b, dout = _inputs(6, 100, "float32", "float32", gpu)
    mean, rstd = kl.layer_norm(x, w, b, stats=True)[1:]
    dx, dw, db = kl.layer_norm_backward(dout, x, mean, rstd, w, b)
    g = torch.Generator().manual_seed(5)
    dirs = [torch.randn(t.shape, generator=g).double().to(gpu) for t in (x, w, b)]
    h = 1e-5

    def loss(s):
        return float((ln64(x.double() + s * dirs[0], w.double() + s * dirs[1], b.double() + s * dirs[2])[0] * dout).sum())

    slope = (loss(h) - loss(-h)) / (2 * h)
    ours = sum(float((d * v.double()).sum()) for d, v in zip(dirs, (dx, dw, db)))
    # fp32 gradients: 1e-5 of the terms; the differences' own error is h^2 of a third derivative of order 1000.
    scale = sum(float((d * v.double()).abs().sum()) for d, v in zip(dirs, (dx, dw, db)))
    assert abs(ours - slope) < 1e-5 * scale + 1e-6


def test_another_stream(gpu):
    import torch

    import kernel_library as kl

    x, w, b, dout = _inputs(2000, 1024, "bfloat16", "bfloat16", gpu)
    y, mean, rstd = kl.layer_norm(x, w, b, stats=True)
    want = kl.layer_norm_backward(dout, x, mean, rstd, w, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(kl.layer_norm_backward(dout, x, mean, rstd, w, b))
    torch.cuda.synchronize()
    for g in got:
        assert all((p == q).all() for p, q in zip(want, g))
