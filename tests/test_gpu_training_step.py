"""A run of the operators together: the training step of a pre-norm MLP block, forward, backward and the orthogonalised
updates, against the same step in 64 bits; and outputs and operands past 32-bit offsets."""

import pytest

from block_oracle import half_step, within
from block_oracle import layer_norm as ln64
from block_oracle import layer_norm_backward as ln_bwd64
from block_oracle import matmul_epilogue as mm64
from block_oracle import matmul_epilogue_backward as mm_bwd64
from block_oracle import newton_schulz as ns64

pytestmark = pytest.mark.gpu


def _block(kl, x, w, dout):
    """y = x + W2 gelu(W1 norm(x) + b1) + b2 and the gradients of x and every parameter; the matrices' updates."""
    import torch

    n, mean, rstd = kl.layer_norm(x, w["gamma"], w["beta"], stats=True)
    pre = torch.empty(x.shape[0], w["W1"].shape[1], dtype=x.dtype, device=x.device)
    h = kl.matmul_epilogue(n, w["W1"], w["b1"], "gelu_tanh", pre=pre)
    y = kl.matmul_epilogue(h, w["W2"], w["b2"], residual=x, rhs_transposed=True)
    g = {}
    dh, g["W2"], g["b2"] = kl.matmul_epilogue_backward(dout, h, w["W2"], bias=w["b2"], rhs_transposed=True)
    dn, g["W1"], g["b1"] = kl.matmul_epilogue_backward(dh, n, w["W1"], "gelu_tanh", pre, w["b1"])
    dx, g["gamma"], g["beta"] = kl.layer_norm_backward(dn, x, mean, rstd, w["gamma"], w["beta"])
    g["x"] = dx + dout
    u = {k: kl.newton_schulz(g[k]) for k in ("W1", "W2")}
    return y, g, u


def _block64(x, w, dout):
    n, mean, rstd = ln64(x, w["gamma"], w["beta"])
    h, pre = mm64(n, w["W1"], w["b1"], "gelu_tanh")
    y, _ = mm64(h, w["W2"], w["b2"], residual=x, rhs_transposed=True)
    g = {}
    dh, g["W2"], g["b2"], _ = mm_bwd64(dout, h, w["W2"], rhs_transposed=True)
    dn, g["W1"], g["b1"], _ = mm_bwd64(dh, n, w["W1"], "gelu_tanh", pre)
    dx, g["gamma"], g["beta"] = ln_bwd64(dn, x, mean, rstd, w["gamma"])
    g["x"] = dx + dout.double()
    return y, g


def _weights(D, H, gpu):
    import torch

    g = torch.Generator().manual_seed(D + H)
    bf = torch.bfloat16
    w = {"gamma": 1 + 0.1 * torch.randn(D, generator=g), "beta": 0.1 * torch.randn(D, generator=g),
         "W1": (torch.randn(D, H, generator=g) / D**0.5).to(bf), "b1": (0.1 * torch.randn(H, generator=g)).to(bf),
         "W2": (torch.randn(D, H, generator=g) / H**0.5).to(bf), "b2": 0.1 * torch.randn(D, generator=g)}
    return {k: v.to(gpu) for k, v in w.items()}


@pytest.mark.parametrize("rows,D,H", [(1, 64, 256), (37, 136, 520), (100, 129, 333), (512, 256, 1024)])
def test_training_step(gpu, rows, D, H):
    """Each tensor between two operators is rounded to bf16 once, 2^-8 at most; a value passes at most 8 of those on its
    way (norm, pre, h, dh, dpre, dn, dx, its own), independent of each other, and no operator steepens a 2-norm error
    by more than 1.13 or spreads it over more than it averages: 8^0.5 * 1.13^2 * 2^-8 of a tensor's 2-norm."""
    import torch

    import kernel_library as kl

    print(f"training step {rows}x{D}x{H}", flush=True)
    w = _weights(D, H, gpu)
    g = torch.Generator().manual_seed(rows)
    x, dout = (torch.randn(rows, D, generator=g).bfloat16().to(gpu) for _ in range(2))
    y, grads, updates = _block(kl, x, w, dout)
    ey, eg = _block64(x, w, dout)
    bound = 8**0.5 * 1.13**2 * half_step(torch.bfloat16)
    for name, a, e in [("y", y, ey)] + [(k, grads[k], eg[k]) for k in eg]:
        assert a.shape == e.shape
        assert float((a.double() - e).norm()) <= bound * float(e.norm()), name
        if name in w:
            assert a.dtype == w[name].dtype
    for k, u in updates.items():
        # The update of the gradient that was computed, not of the exact one (it turns small singular values up).
        e = ns64(grads[k])
        assert float((u.double() - e).norm()) <= (half_step(torch.bfloat16) + 3 * 2.0**-18 * 700) * float(e.norm())


def test_training_step_in_a_graph_between_eager_ones(gpu):
    """Captured once and replayed with eager steps of other inputs between the replays, and beside a second graph."""
    import torch

    import kernel_library as kl

    rows, D, H = 260, 256, 1024  # (the weights' gradients contract over 260 rows: whole and partial K tiles)
    w = _weights(D, H, gpu)
    x, dout = (torch.randn(rows, D, device=gpu).bfloat16() for _ in range(2))
    _block(kl, x, w, dout)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _block(kl, x, w, dout)
        graphs.append((graph, out))
    other = torch.randn(3 * rows, D, device=gpu).bfloat16()
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        dout.copy_(torch.randn_like(dout))
        y, grads, updates = _block(kl, x, w, dout)
        for graph, out in graphs:
            _block(kl, other, w, other)
            graph.replay()
            torch.cuda.synchronize()
            assert (out[0] == y).all()
            assert all((out[1][k] == grads[k]).all() for k in grads)
            assert all((out[2][k] == updates[k]).all() for k in updates)


def test_threads_at_once(gpu):
    """Calls from several threads, each on its own stream, give what they give alone."""
    import threading

    import torch

    import kernel_library as kl

    jobs = []
    for i, (rows, D, H) in enumerate([(100, 136, 264), (64, 256, 512), (33, 129, 200), (200, 64, 128)]):
        w = _weights(D, H, gpu)
        g = torch.Generator().manual_seed(i)
        x, dout = (torch.randn(rows, D, generator=g).bfloat16().to(gpu) for _ in range(2))
        jobs.append((x, w, dout, _block(kl, x, w, dout)))
    torch.cuda.synchronize()
    wrong = []

    def work(job):
        x, w, dout, want = job
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                y, grads, updates = _block(kl, x, w, dout)
                stream.synchronize()
                if not ((y == want[0]).all() and all((grads[k] == want[1][k]).all() for k in grads)
                        and all((updates[k] == want[2][k]).all() for k in updates)):
                    wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rows_past_32_bit_offsets(gpu):
    """4.5 GiB of rows: the last ones are where they belong."""
    import torch

    import kernel_library as kl

    rows, D = 73000, 32768
    x = torch.empty(rows, D, dtype=torch.bfloat16, device=gpu)
    x.normal_()
    w = torch.randn(D, device=gpu).bfloat16()
    y, mean, rstd = kl.layer_norm(x, w, stats=True)
    for at in (0, 36000, rows - 3):
        e, em, er = ln64(x[at:at + 3], w)
        within(y[at:at + 3], e, 2.0**-7 * e.abs() + 1e-4)
        within(mean[at:at + 3], em, 1e-6)
    got = kl.layer_norm_backward(y, x, mean, rstd, w, w)
    for at in (0, rows - 3):
        e = ln_bwd64(y[at:at + 3], x[at:at + 3], mean[at:at + 3], rstd[at:at + 3], w)[0]
        within(got[0][at:at + 3], e, 2.0**-7 * e.abs() + 1e-3 * float(e.abs().max()))
    sums = torch.zeros(D, dtype=torch.float64, device=gpu)
    mags = torch.zeros(D, dtype=torch.float64, device=gpu)
    for at in range(0, rows, 4000):
        part = y[at:at + 4000].double()
        sums += part.sum(0)
        mags += part.abs().sum(0)
    within(got[2], sums, 2.0**-8 * sums.abs() + 700 * 2.0**-24 * mags)


def test_an_output_past_32_bit_offsets(gpu):
    import torch

    import kernel_library as kl

    M, N, K = 73000, 32768, 8
    for transposed in (False, True):
        lhs = torch.randn(M, K, device=gpu).bfloat16()
        rhs = torch.randn(*((N, K) if transposed else (K, N)), device=gpu).bfloat16()
        bias = torch.randn(N, device=gpu).bfloat16()
        out = kl.matmul_epilogue(lhs, rhs, bias, "relu", rhs_transposed=transposed)
        for at in (0, 65500, M - 40):
            e = mm64(lhs[at:at + 40], rhs, bias, "relu", rhs_transposed=transposed)[0]
            within(out[at:at + 40], e, 2.0**-8 * e.abs() + 1e-4)
