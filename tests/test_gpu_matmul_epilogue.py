"""matmul_epilogue and its gradients against their plain 64-bit forms."""

import itertools

import pytest

from block_oracle import ACTIVATIONS, half_step, within
from block_oracle import matmul_epilogue as mm64
from block_oracle import matmul_epilogue_backward as mm_bwd64
from block_oracle import matmul_epilogue_tolerance as mm_tol

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (16, 64, 64), (17, 33, 65), (32, 136, 72), (65, 129, 100), (128, 128, 128),
          (130, 264, 320), (1, 1501, 777), (7, 2000, 1504), (257, 513, 200), (300, 100, 1000), (520, 640, 64)]


def _inputs(M, N, K, gpu, transposed=False, bias="bfloat16", residual=True, seed=0):
    import torch

    g = torch.Generator().manual_seed(M * 7919 + N * 31 + K + seed)
    lhs = torch.randn(M, K, generator=g).bfloat16()
    rhs = (torch.randn(*((N, K) if transposed else (K, N)), generator=g) / max(1, K) ** 0.5).bfloat16()
    b = torch.randn(N, generator=g).to(getattr(torch, bias)) if bias else None
    r = torch.randn(M, N, generator=g).bfloat16() if residual else None
    return [t.to(gpu) if t is not None else None for t in (lhs, rhs, b, r)]


def _check(lhs, rhs, b, act, r, transposed, out, pre=None):
    e, epre = mm64(lhs, rhs, b, act, r, transposed)
    within(out, e, mm_tol(lhs, rhs, e, b, r, transposed))
    if pre is not None:
        within(pre, epre, mm_tol(lhs, rhs, epre, b, None, transposed))


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_shapes(gpu, M, N, K, transposed):
    import torch

    import kernel_library as kl

    print(f"matmul_epilogue {M}x{N}x{K} {transposed}", flush=True)
    lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
    pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
    out = kl.matmul_epilogue(lhs, rhs, b, "silu", r, rhs_transposed=transposed, pre=pre)
    _check(lhs, rhs, b, "silu", r, transposed, out, pre)
    _check(lhs, rhs, None, "none", None, transposed, kl.matmul_epilogue(lhs, rhs, rhs_transposed=transposed))


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (1, 9, 1000), (2, 4097, 71), (31, 129, 65), (32, 128, 127), (33, 8, 9),
                                   (40, 1001, 2049), (64, 65, 4099), (100, 200, 201), (256, 300, 333), (257, 300, 333),
                                   (600, 77, 90), (5, 7, 100), (5, 100, 7), (9, 2051, 2049)])
def test_odd_sizes_as_they_are_and_copied(gpu, M, N, K, transposed):
    """Rows that do not start on 16 bytes: few of them go through registers (whole and partial pieces, tiles and parts),
    more are copied to padded ones; aligned sizes at odd addresses too, and infinities that must not leave the last
    piece."""
    import torch

    import kernel_library as kl

    print(f"matmul_epilogue {M}x{N}x{K} {transposed}", flush=True)
    for off in (0, 1, 3):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed, "float32")

        def at(t):
            big = torch.full((t.numel() + 64,), float("inf"), dtype=t.dtype, device=gpu)
            view = big[16 + off:16 + off + t.numel()].view(t.shape)
            view.copy_(t)
            return view

        out = kl.matmul_epilogue(at(lhs), at(rhs), b, "silu", at(r), rhs_transposed=transposed)
        _check(lhs, rhs, b, "silu", r, transposed, out)
        pre = r
        got = kl.matmul_epilogue_backward(at(r), at(lhs), at(rhs), "silu", at(pre), b, rhs_transposed=transposed)
        _check_backward(r, lhs, rhs, "silu", pre, transposed, *got)


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("bias,residual", [("", False), ("bfloat16", False), ("float32", True), ("", True)])
def test_epilogues(gpu, act, bias, residual):
    import torch

    import kernel_library as kl

    for (M, N, K), transposed in itertools.product([(70, 200, 136), (33, 77, 40)], (False, True)):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed, bias, residual)
        rhs *= 3  # activations over their whole range
        pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
        out = kl.matmul_epilogue(lhs, rhs, b, act, r, rhs_transposed=transposed, pre=pre)
        _check(lhs, rhs, b, act, r, transposed, out, pre)
        again = kl.matmul_epilogue(lhs, rhs, b, None if act == "none" else act, r, rhs_transposed=transposed)
        assert (again == out).all()


def _configs():
    from kernel_library.config import TileConfig

    found = [(256, 256, 64, 8, 2, 0), (256, 128, 64, 8, 3, 0), (128, 256, 64, 8, 3, 0), (128, 128, 64, 4, 4, 0),
             (64, 128, 64, 4, 3, 0), (128, 64, 64, 4, 3, 0), (64, 64, 64, 4, 2, 0), (64, 64, 64, 4, 4, 0),
             (32, 128, 64, 4, 4, 1), (128, 128, 64, 4, 3, 1)]
    return [TileConfig(bm, bn, bk, w, s, 1, 8, v) for bm, bn, bk, w, s, v in found]


@pytest.mark.parametrize("cfg", _configs(), ids=lambda c: c.name)
def test_every_config_and_split(gpu, cfg):
    import dataclasses

    import kernel_library as kl

    assert cfg in kl.epilogue_configs()
    for (M, N, K), transposed in itertools.product([(300, 392, 1000), (261, 515, 200)], (False, True)):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
        for parts in (1, 2, 4):
            c = dataclasses.replace(cfg, split_k=parts, group_m=3 if parts == 2 else 8)
            print(f"{c.name} {M}x{N}x{K} {transposed}", flush=True)
            out = kl.matmul_epilogue(lhs, rhs, b, "gelu", r, rhs_transposed=transposed, cfg=c)
            _check(lhs, rhs, b, "gelu", r, transposed, out)


@pytest.mark.parametrize("transposed", [False, True])
def test_sixteen_parts_of_a_long_contraction(gpu, transposed):
    import dataclasses

    import kernel_library as kl

    lhs, rhs, b, r = _inputs(40, 136, 5000, gpu, transposed)
    c = dataclasses.replace(_configs()[-2], split_k=16)
    _check(lhs, rhs, b, "relu", r, transposed, kl.matmul_epilogue(lhs, rhs, b, "relu", r, transposed, cfg=c))


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("M,N,K", [(0, 8, 8), (8, 0, 8), (5, 9, 0), (0, 0, 0), (1, 16, 0)])
def test_empty_sizes(gpu, M, N, K, transposed):
    import torch

    import kernel_library as kl

    lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
    pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
    out = kl.matmul_epilogue(lhs, rhs, b, "gelu", r, rhs_transposed=transposed, pre=pre)
    _check(lhs, rhs, b, "gelu", r, transposed, out, pre)
    dout = torch.randn(M, N, device=gpu).bfloat16()
    dlhs, drhs, db = kl.matmul_epilogue_backward(dout, lhs, rhs, "gelu", pre, b, rhs_transposed=transposed)
    assert dlhs.shape == lhs.shape and drhs.shape == rhs.shape and db.shape == b.shape
    e = mm_bwd64(dout, lhs, rhs, "gelu", pre, transposed)
    assert (dlhs == 0).all() and (drhs == 0).all()
    within(db, e[2], 2.0**-8 * e[2].abs() + 1e-5 * (dout.double().abs().sum(0)))


def test_what_lies_around_operands_and_outputs(gpu):
    """NaN next to every operand reaches no output, and nothing next to an output is written."""
    import torch

    import kernel_library as kl

    for (M, N, K), transposed, off in itertools.product([(33, 72, 40), (30, 61, 51), (130, 264, 200)], (False, True), (0, 1, 8)):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
        dout = torch.randn(M, N, device=gpu).bfloat16()

        def inside(t, value=float("nan")):
            big = torch.full((t.numel() + 4096 + off,), value, dtype=t.dtype, device=gpu)
            at = 2048 + off
            view = big[at:at + t.numel()].view(t.shape)
            view.copy_(t)
            return big, view

        (_, lhs2), (_, rhs2), (_, b2), (_, r2), (_, d2) = (inside(t) for t in (lhs, rhs, b, r, dout))
        big_o, out = inside(torch.zeros_like(r), 7.0)
        big_p, pre = inside(torch.zeros_like(r), 7.0)
        kl.matmul_epilogue(lhs2, rhs2, b2, "gelu_tanh", r2, rhs_transposed=transposed, pre=pre, out=out)
        _check(lhs, rhs, b, "gelu_tanh", r, transposed, out, pre)
        for big in (big_o, big_p):
            assert (big[:2048 + off] == 7).all() and (big[2048 + off + M * N:] == 7).all()
        got = kl.matmul_epilogue_backward(d2, lhs2, rhs2, "gelu_tanh", pre, b2, rhs_transposed=transposed)
        _check_backward(dout, lhs, rhs, "gelu_tanh", pre, transposed, *got)


def test_infinities_stay_in_their_rows_and_columns(gpu):
    import torch

    import kernel_library as kl

    for transposed, (M, N, K) in itertools.product((False, True), [(64, 136, 72), (70, 131, 33)]):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
        lhs[3, K - 1] = float("inf")
        r[5, N - 1] = float("nan")
        b[N - 2] = float("-inf")
        out = kl.matmul_epilogue(lhs, rhs, b, "relu", r, rhs_transposed=transposed)
        e = mm64(lhs, rhs, b, "relu", r, transposed)[0]
        tol = torch.nan_to_num(mm_tol(lhs, rhs, e, b, r, transposed), nan=0.0, posinf=0.0)
        within(out, e, tol)


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_over_all_of_bf16(gpu, act):
    """Every finite bf16 value and the infinities through the epilogue (an empty product and a residual of 0) and, as pre,
    through the gradient's column sums.

    The values: an exponential of argument a is off by 2^-24 a (a up to 100 before the result underflows), the rest by
    a few 2^-24: 2^-17 in all, relative, down to where fp32 itself ends: the hardware's reciprocal gives 0 where its result
    is under 2^-126, which happens to a sigmoid left of -87.3, and a double's exponential has the sigmoid under 2^-150
    (nothing of it left in fp32) left of -104, so what is lost is under 104 * 2^-126 = 1.23e-36."""
    import torch

    import kernel_library as kl
    from block_oracle import act as act64
    from block_oracle import act_slope

    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).to(gpu)
    x = x[torch.isfinite(x)]
    n = x.numel()
    out = kl.matmul_epilogue(torch.empty(1, 0, dtype=torch.bfloat16, device=gpu),
                             torch.empty(0, n, dtype=torch.bfloat16, device=gpu), x, act)
    e = act64(act, x.double())
    e = torch.where(x.double() < -1e10, torch.zeros_like(e), e) if act != "relu" else e  # 0 times infinity in the formula
    e = torch.where(x.double() > 1e10, x.double(), e)
    within(out[0], e, (2.0**-17 + half_step(torch.bfloat16)) * e.abs() + 104 * 2.0**-126)
    one = torch.ones(1, n, dtype=torch.bfloat16, device=gpu)
    bias = torch.empty(n, device=gpu)
    db = kl.matmul_epilogue_backward(one, torch.empty(1, 0, dtype=torch.bfloat16, device=gpu),
                                     torch.empty(0, n, dtype=torch.bfloat16, device=gpu), act, x[None], bias)[2]
    far = x.double().abs() > 1e4
    e = act_slope(act, torch.where(far, torch.sign(x.double()) * 1e4, x.double()))
    # Near the zero of a slope its two terms cancel: they are off by 2^-17 of the larger, under 1.2.
    within(db, e, 2.0**-16 * torch.maximum(e.abs(), torch.full_like(e, 1e-2)))


def _check_backward(dout, lhs, rhs, act, pre, transposed, dlhs, drhs, db):
    """dpre is rounded to bf16 for the products, each gradient once more.

    An element of a product is off by at most 2^-8 of the sum of its terms' magnitudes (and 2^-23 K of it for fp32
    sums), and over a whole gradient the roundings are independent: their 2-norm is under 2^-8 of the result's, the
    dpre's and the output's together 2^-8 sqrt(2) at the very most of half a step each."""
    import torch

    e_lhs, e_rhs, e_b, dpre = mm_bwd64(dout, lhs, rhs, act, pre, transposed)
    w = rhs.double().abs().t().contiguous() if transposed else rhs.double().abs()
    mag_l = dpre.abs() @ w.t().contiguous()
    mag_r = lhs.double().abs().t().contiguous() @ dpre.abs()
    mag_r = mag_r.t().contiguous() if transposed else mag_r
    M, N = dout.shape
    slope = dout.double().abs().sum(0)
    for got, e, mag, n in ((dlhs, e_lhs, mag_l, N), (drhs, e_rhs, mag_r, M)):
        if got is None:
            continue
        rounded = half_step(torch.bfloat16)
        within(got, e, (rounded * (1 + rounded) + (n + 2) * 2.0**-23 + 2.0**-16) * mag + rounded * e.abs() + 1e-30)
        if e.numel() > 1000 and float(e.norm()) > 0:
            assert float((got.double() - e).norm() / e.norm()) < 2.0**-8 * 2**0.5
    if db is not None:
        within(db, e_b, ((M + 20) * 2.0**-24 + 2.0**-16) * slope * 1.2 + half_step(db.dtype) * e_b.abs())


@pytest.mark.parametrize("act", ["none", "gelu", "relu"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gradients(gpu, M, N, K, transposed, act):
    import torch

    import kernel_library as kl

    print(f"matmul_epilogue_backward {M}x{N}x{K} {transposed} {act}", flush=True)
    lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed, "float32")
    dout = r
    pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
    kl.matmul_epilogue(lhs, rhs, b, act, rhs_transposed=transposed, pre=pre)
    got = kl.matmul_epilogue_backward(dout, lhs, rhs, act, pre, b, rhs_transposed=transposed)
    assert got[0].shape == lhs.shape and got[1].shape == rhs.shape and got[2].dtype == torch.float32
    _check_backward(dout, lhs, rhs, act, pre, transposed, *got)
    for need_l, need_r, bias in ((True, False, None), (False, True, None), (False, False, b.bfloat16())):
        part = kl.matmul_epilogue_backward(dout, lhs, rhs, act, pre, bias, transposed, need_l, need_r)
        assert (part[0] is None) != need_l and (part[1] is None) != need_r and (part[2] is None) == (bias is None)
        if need_l:
            assert (part[0] == got[0]).all()
        if need_r:
            assert (part[1] == got[1]).all()
        if bias is not None:
            _check_backward(dout, lhs, rhs, act, pre, transposed, None, None, part[2])


def test_gradient_against_differences(gpu):
    """The directional derivative of the 64-bit forward form, by central differences."""
    import torch

    import kernel_library as kl

    for act, transposed in itertools.product(("gelu", "gelu_tanh", "silu"), (False, True)):
        lhs, rhs, b, r = _inputs(24, 40, 56, gpu, transposed, "float32")
        pre = mm64(lhs, rhs, b, act, None, transposed)[1].bfloat16()
        dlhs, drhs, db = kl.matmul_epilogue_backward(r, lhs, rhs, act, pre, b, rhs_transposed=transposed)
        g = torch.Generator().manual_seed(3)
        dirs = [torch.randn(t.shape, generator=g).double().to(gpu) for t in (lhs, rhs, b)]
        h = 1e-5

        def loss(s):
            return float((mm64(lhs.double() + s * dirs[0], rhs.double() + s * dirs[1], b.double() + s * dirs[2], act, None,
                               transposed)[0] * r.double()).sum())

        slope = (loss(h) - loss(-h)) / (2 * h)
        ours = sum(float((d * v.double()).sum()) for d, v in zip(dirs, (dlhs, drhs, db)))
        # Each product of a direction and a gradient is off by a few bf16 roundings (pre's, dpre's, its own), independent.
        scale = sum(float((d * v.double()).square().sum()) for d, v in zip(dirs, (dlhs, drhs, db))) ** 0.5
        assert abs(ours - slope) < 8 * 3 * 2.0**-8 * scale


def test_same_bits_on_streams_and_in_graphs(gpu):
    import torch

    import kernel_library as kl

    # Split-K, padded operands and the plain path, forward and backward.
    for M, N, K, transposed in ((40, 520, 2048, False), (70, 131, 333, True), (512, 512, 256, False), (4096, 128, 136, False),
                                (4095, 129, 128, True)):
        lhs, rhs, b, r = _inputs(M, N, K, gpu, transposed)
        pre = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)

        def step():
            out = kl.matmul_epilogue(lhs, rhs, b, "silu", r, rhs_transposed=transposed, pre=pre)
            return (out, *kl.matmul_epilogue_backward(r, lhs, rhs, "silu", pre, b, rhs_transposed=transposed))

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.synchronize()
        assert all((p == q).all() for p, q in zip(want, other))
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs = step()
            graphs.append((graph, outs))
        for k in range(3):
            lhs.copy_(_inputs(M, N, K, gpu, transposed, seed=k + 1)[0])
            want = step()
            torch.cuda.synchronize()
            for graph, outs in graphs:
                graph.replay()
                torch.cuda.synchronize()
                assert all((p == q).all() for p, q in zip(want, outs))
