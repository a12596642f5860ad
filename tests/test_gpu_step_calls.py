"""Calls of the 8-bit step's operators that the documentation allows and nothing else here makes: expanded operands and
scales, outputs of more than 2^20 columns, long products, very tall matrices, modes of torch."""

import pytest

from block_oracle import half_step, within
from step_oracle import quantize as q64
from step_oracle import residual_norm as rn64
from test_gpu_fp8 import _check_product, _operands, _rows, _same_values
from test_gpu_residual_norm import TYPES, _check_backward, _check_forward, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(70, 90, 300), (4100, 1030, 2176)])
def test_expanded_operands_and_scales(gpu, M, N, K):
    """Every row the same, and one scale for all of an operand, by strides of 0 (at a size whose scales are turned too)."""
    import torch

    import kernel_library as kl

    lhs, ls, rhs, rs = _operands(M, N, K, "e4m3", "float32", False, gpu)
    one = lhs[:1].expand(M, K), ls[:1].expand(M, -1)
    out = kl.matmul_fp8(*one, rhs, rs)
    assert torch.equal(out, kl.matmul_fp8(lhs[:1].repeat(M, 1), ls[:1].repeat(M, 1), rhs, rs))
    assert torch.equal(out, out[:1].expand(M, N))
    exponent = torch.full((1, 1), 125, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu)
    for scale in (torch.full((1, 1), 0.25, device=gpu), exponent):
        s, t = (scale.expand(n, -(-K // 128)) for n in (M, N))
        out = kl.matmul_fp8(lhs, s, rhs, t)
        assert torch.equal(out, kl.matmul_fp8(lhs, s.contiguous(), rhs, t.contiguous()))
        if M < 1000:
            _check_product(out, lhs, s, rhs, t)


@pytest.mark.parametrize("scales,square", [("float32", True), ("float32", False), ("e8m0", True)])
@pytest.mark.parametrize("M,N,K", [(3, (1 << 20) + 24, 200), (3, (1 << 20) + 13, 130), ((1 << 20) + 5, 9, 136)])
def test_more_than_2_to_the_20_columns_or_rows(gpu, M, N, K, scales, square):
    import kernel_library as kl

    lhs, ls, rhs, rs = _operands(M, N, K, "e4m3", scales, square, gpu)
    out = kl.matmul_fp8(lhs, ls, rhs, rs)
    for cut in (slice(0, 300), slice(-300, None)):
        if N > M:
            first = range(N)[cut][0]
            at = slice(first // 128 * 128, range(N)[cut][-1] + 1)
            r = rs[at.start // 128:] if square and cut.start else rs[:-(-at.stop // 128)] if square else rs[at]
            _check_product(out[:, at].contiguous(), lhs, ls, rhs[at], r)
        else:
            _check_product(out[cut], lhs[cut], ls[cut], rhs, rs)


@pytest.mark.parametrize("scales,square", [("float32", True), ("float32", False), ("e8m0", False)])
def test_long_products(gpu, scales, square):
    """65537 K tiles, the last of one value: small whole numbers in few places, whose sums are exact in fp32."""
    import torch

    import kernel_library as kl

    M, N, K = 3, 5, (1 << 23) + 1
    g = torch.Generator().manual_seed(0)
    kb = -(-K // 128)
    rhs = torch.randint(-2, 3, (N, K), generator=g, dtype=torch.int8)
    lhs = torch.zeros(M, K, dtype=torch.int8)
    for r in range(M):
        lhs[r, torch.randint(K, (60,), generator=g)] = 3
        lhs[r, torch.tensor([0, 127 + r, K // 2, K - 2 - r, K - 1])] = 1
    ls, rs = (torch.exp2(torch.randint(-1, 2, (n, kb), generator=g).float()) for n in (M, 1 if square else N))
    wide = [t.repeat_interleave(128, 1)[:, :K] for t in (ls, rs)]
    e = (lhs.double() * wide[0].double()) @ (rhs.double() * wide[1].double()).t()
    if scales == "e8m0":
        ls, rs = ((127 + t.log2()).to(torch.uint8).view(torch.float8_e8m0fnu) for t in (ls, rs))
    lhs, rhs = (t.float().to(torch.float8_e4m3fn).to(gpu) for t in (lhs, rhs))
    for cfg in (None, *kl.fp8_configs()):
        out = kl.matmul_fp8(lhs, ls.to(gpu), rhs, rs.to(gpu), cfg=cfg)
        assert torch.equal(out.cpu(), e.bfloat16()), cfg


def test_a_very_tall_matrix(gpu):
    """2^26 rows of 3 values: their transpose has 2^19 blocks a row."""
    import torch

    import kernel_library as kl

    M, K = (1 << 26) + 3, 3
    x = torch.randn(M, K, device=gpu).bfloat16()
    q, s, q_t, s_t = kl.quantize_fp8(x, transposed=True)
    for cut in (slice(0, 256), slice(M // 2 // 128 * 128, M // 2 // 128 * 128 + 256), slice(M // 128 * 128, None)):
        eq, es = q64(x[cut])
        _same_values(q[cut], eq)
        _same_values(s[cut], es)
        eq, es = q64(x[cut].t().contiguous())
        _same_values(q_t[:, cut], eq)
        first = cut.start // 128
        _same_values(s_t[:, first:first + es.shape[1]], es)


@pytest.mark.parametrize("M,N,K", [(257, 300, 520), (1000, 70, 33)])
def test_gradients_of_rows_that_are_apart(gpu, M, N, K):
    """The output's gradient, its operands and their scales as views of wider memory: the same bits."""
    import torch

    import kernel_library as kl

    dout = _rows(M, N, 5, gpu).bfloat16()
    lt, lts = kl.quantize_fp8(_rows(K, M, 6, gpu))
    rt, rts = kl.quantize_fp8(_rows(K, N, 7, gpu), (128, 128))
    first = kl.matmul_fp8_backward(dout, lt, lts, rt, rts)

    def apart(t, at):
        wide = torch.full((t.shape[0], t.shape[1] + 37), 0x7F, dtype=torch.uint8, device=gpu).view(t.dtype) \
            if t.element_size() == 1 else torch.full((t.shape[0], t.shape[1] + 37), torch.nan, dtype=t.dtype, device=gpu)
        bits = torch.uint8 if t.element_size() == 1 else t.dtype
        wide.view(bits)[:, at:at + t.shape[1]] = t.contiguous().view(bits)
        return wide[:, at:at + t.shape[1]]

    for at in (0, 1, 16):
        got = kl.matmul_fp8_backward(apart(dout, at), apart(lt, at), apart(lts, at), apart(rt, at), apart(rts, at))
        assert all(torch.equal(u, v) for u, v in zip(first, got)), at
        for kw in (dict(need_dlhs=False), dict(need_drhs=False)):
            one = kl.matmul_fp8_backward(apart(dout, at), apart(lt, at), apart(lts, at), apart(rt, at), apart(rts, at), **kw)
            assert all(torch.equal(u, v) for u, v in zip(first, one) if v is not None), (at, kw)


@pytest.mark.parametrize("D", [5, 264, 9000])
def test_rows_that_are_all_the_same(gpu, D):
    """Operands with a row stride of 0, in the norm and its gradients."""
    import torch

    import kernel_library as kl

    a, dy, dh = _inputs(1, 50, D, TYPES[1], "shared", True, gpu)
    a["x"], dy, dh = (t[0, :1].expand(50, D) for t in (a["x"], dy, dh))
    a["residual"] = a["residual"][0]
    y, hidden, rstd, post_rstd = kl.residual_norm(stats=True, **a)
    _check_forward(a, 1.0, 1e-6, y, hidden, rstd, post_rstd)
    got = kl.residual_norm_backward(dy, dh, a["x"], hidden, rstd, a["weight"], a["gate"], 1.0, post_rstd, a["post_weight"])
    _check_backward(a, 1.0, dy, dh, hidden, rstd, post_rstd, got)
    v, w = a["x"][0], a["residual"][0]  # one row, of one dimension
    y, hidden = kl.residual_norm(v, w, a["weight"])
    e = rn64(v, w, a["weight"])
    assert y.shape == (D,) and torch.equal(hidden, (v.float() + w.float()).to(w.dtype))
    within(y, e[0], (half_step(y.dtype) + 128 * 2.0**-24) * e[0].abs() + 2.0**-24 * e[0].abs())


@pytest.mark.parametrize("mode", ["inference_mode", "autocast", "no_grad"])
def test_modes(gpu, mode):
    import torch

    import kernel_library as kl

    x, res = torch.randn(40, 264, device=gpu).bfloat16(), torch.randn(40, 264, device=gpu)
    w = torch.nn.Parameter(torch.ones(264, device=gpu))
    dout = torch.randn(40, 96, device=gpu).bfloat16()

    def step(weight):
        y, hidden, rstd, _ = kl.residual_norm(x, res, weight, stats=True)
        a, b = kl.quantize_fp8(y, transposed=True), kl.quantize_fp8(res[:32].repeat(3, 1), (128, 128), transposed=True)
        dy, dw = kl.matmul_fp8_backward(dout, *a[2:], *b[2:])
        norm, clipped = kl.clip_grad_norm([dy, dw], 0.1)
        return (y, hidden, kl.matmul_fp8(*a[:2], *b[:2]), dy, dw, norm, *clipped,
                *kl.residual_norm_backward(dy, None, x, hidden, rstd, weight)[:3])

    first = step(w.detach())
    context = {"inference_mode": torch.inference_mode, "no_grad": torch.no_grad,
               "autocast": lambda: torch.autocast("cuda", torch.bfloat16)}[mode]
    with context():
        got = step(w.detach() if mode == "autocast" else w)
        assert all(not t.requires_grad for t in got)
    assert all(torch.equal(u, v) for u, v in zip(first, got))


def test_infinite_norms(gpu):
    import torch

    import kernel_library as kl

    g = [torch.randn(3000, device=gpu), torch.randn(70, device=gpu).bfloat16()]
    norm, clipped = kl.clip_grad_norm(g, float("inf"))
    assert torch.isfinite(norm) and all(torch.equal(a, b) for a, b in zip(g, clipped))
    g[0][5] = float("inf")
    norm, clipped = kl.clip_grad_norm(g, 1.0)
    assert torch.isinf(norm) and not clipped[1].any()
    norm, clipped = kl.clip_grad_norm(g, float("inf"))
    assert torch.isinf(norm) and all(torch.isnan(c).all() for c in clipped)
    # Squares beyond fp32 whose sum is not: the norm itself leaves fp32.
    norm, clipped = kl.clip_grad_norm([torch.full((100,), 3e38, device=gpu)], 1.0)
    assert torch.isinf(norm) and not clipped[0].any()


@pytest.mark.parametrize("eps", [1e-6, 1e-35, 0.0])
@pytest.mark.parametrize("D", [1, 3, 4, 8, 40, 100, 250, 500, 1000, 3000, 8000, 12000, 20000])
def test_rows_of_every_magnitude(gpu, D, eps):
    """Rows whose squares leave fp32 beside ordinary ones, several to a wave: each as if by itself.  Then infinities and
    NaN in some of them: the others, and their gradients, keep their bits."""
    import torch

    import kernel_library as kl

    g = torch.Generator().manual_seed(D)
    rows = 50
    scale = torch.exp2(torch.randint(-100, 100, (rows, 1), generator=g).float())
    scale[::4] = 1.0
    x = (torch.randn(rows, D, generator=g) * scale).to(gpu)
    res = (torch.randn(rows, D, generator=g) * scale.flip(0)).to(gpu)
    x[x.abs() < 1e-32], res[res.abs() < 1e-32] = 1e-32, 1e-32  # (no row of zeros without an eps, nothing subnormal)
    w = (1 + torch.rand(D, generator=g)).to(gpu)
    a = dict(x=x, residual=res, weight=w, gate=None, post_norm=True, post_weight=w)
    y, hidden, rstd, post_rstd = kl.residual_norm(eps=eps, stats=True, **a)
    _check_forward(a, 1.0, eps, y, hidden, rstd, post_rstd)
    dy, dh = (torch.randn(rows, D, generator=g).to(gpu) for _ in range(2))
    first = kl.residual_norm_backward(dy, dh, x, hidden, rstd, w, None, 1.0, post_rstd, w)
    bad = torch.zeros(rows, dtype=torch.bool, device=gpu)
    bad[torch.tensor([1, 7, 8, 30])] = True
    z, r = x.clone(), res.clone()
    z[1, D // 2], r[7, 0], z[8, D - 1], r[30, D // 3] = float("nan"), float("inf"), float("-inf"), float("nan")
    y2, hidden2, rstd2, post2 = kl.residual_norm(eps=eps, stats=True, **(a | dict(x=z, residual=r)))
    for u, v in ((y, y2), (hidden, hidden2), (rstd, rstd2), (post_rstd, post2)):
        assert torch.equal(u[~bad], v[~bad])
    assert torch.isnan(y2[bad]).any(-1).all()
    got = kl.residual_norm_backward(dy, dh, z, hidden2, rstd2, w, None, 1.0, post2, w)
    for u, v in zip(first[:2], got[:2]):
        assert torch.equal(u[~bad], v[~bad])
