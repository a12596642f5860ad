"""The native calls of the operators (csrc/host/mi_operator_call.cpp): they take ordinary calls, answer as the Python
bodies do, and leave everything else to them."""

import pytest

pytestmark = pytest.mark.gpu


class _Python:
    """The extension with its operators left to the Python bodies."""

    def __init__(self, native):
        self.native = native

    def __getattr__(self, name):
        if name in ("layer_norm", "layer_norm_backward", "matmul_epilogue", "matmul_epilogue_backward", "newton_schulz"):
            return lambda *args: None
        return getattr(self.native, name)


def _both(monkeypatch, call):
    """``call()`` by the native functions and by the Python bodies."""
    from kernel_library import _operands, epilogue, norm, orthogonal

    call()  # binds
    native = _operands._torch_call
    assert native.knows_operators()
    fast = call()
    with monkeypatch.context() as m:
        for mod in (epilogue, norm, orthogonal):
            m.setattr(mod, "_torch_call", _Python(native))
        slow = call()
    return fast, slow


def _same(a, b):
    if isinstance(a, (tuple, list)):
        return type(a) is type(b) and len(a) == len(b) and all(_same(x, y) for x, y in zip(a, b))
    if a is None or b is None:
        return a is b
    return a.dtype == b.dtype and a.shape == b.shape and not a.requires_grad and bool((a == b).all())


def test_answers_are_the_python_bodies(gpu, monkeypatch):
    import torch

    import kernel_library as kl

    bf = torch.bfloat16
    x, w, b = (torch.randn(s, device=gpu).to(bf) for s in ((3, 5, 320), (320,), (320,)))
    lhs, rhs = torch.randn(70, 96, device=gpu).to(bf), torch.randn(96, 136, device=gpu).to(bf)
    bias, res, pre = torch.randn(136, device=gpu), torch.randn(70, 136, device=gpu).to(bf), torch.zeros(70, 136, device=gpu).to(bf)
    param = torch.nn.Parameter(rhs)
    y, mean, rstd = kl.layer_norm(x, w, b, stats=True)
    calls = [
        lambda: kl.layer_norm(x),
        lambda: kl.layer_norm(x, w, b, 1e-3),
        lambda: kl.layer_norm(x, w.float(), stats=True),
        lambda: kl.layer_norm(x, w, b, out=torch.zeros_like(x)),
        lambda: kl.layer_norm_backward(y, x, mean, rstd, w, b),
        lambda: kl.layer_norm_backward(y, x, mean, rstd, None, b, need_dx=False),
        lambda: kl.matmul_epilogue(lhs, param),
        lambda: kl.matmul_epilogue(lhs, rhs, bias, "gelu", res, pre=pre),
        lambda: kl.matmul_epilogue(lhs, rhs.t().contiguous(), bias.to(bf), "silu", rhs_transposed=True, out=torch.zeros_like(res)),
        lambda: kl.matmul_epilogue_backward(res, lhs, param, "gelu", pre, bias),
        lambda: kl.matmul_epilogue_backward(res, lhs, rhs, need_dlhs=False),
        lambda: kl.newton_schulz(lhs),
        lambda: kl.newton_schulz(x.float(), steps=2, coefficients=(1.5, -0.5, 0.0), eps=0.0, out=torch.zeros_like(x)),
    ]
    for i, call in enumerate(calls):
        fast, slow = _both(monkeypatch, call)
        assert _same(fast, slow), i


def test_ordinary_calls_are_taken(gpu):
    import torch

    import kernel_library as kl
    from kernel_library import _operands

    t = torch.randn(16, 64, device=gpu).bfloat16()
    kl.layer_norm(t[:, :8])  # the Python body binds
    n = _operands._torch_call
    assert n.layer_norm(t, None, None, 1e-5, None, False) is not None
    assert n.matmul_epilogue(t, t, None, 0, None, True, None, None) is not None
    assert n.newton_schulz(t, 5, 3.4445, -4.775, 2.0315, 1e-7, None) is not None
    # Left to the Python body: another layout, type, device, an overlap, nothing to do.
    assert n.layer_norm(t[:, :8], None, None, 1e-5, None, False) is None
    assert n.layer_norm(t.double(), None, None, 1e-5, None, False) is None
    assert n.layer_norm(t.cpu(), None, None, 1e-5, None, False) is None
    assert n.layer_norm(t, None, None, 1e-5, t, False) is None
    assert n.layer_norm(t, None, None, -1.0, None, False) is None
    assert n.layer_norm(t, t[0, :8], None, 1e-5, None, False) is None
    assert n.layer_norm(t[:0], None, None, 1e-5, None, False) is None
    assert n.matmul_epilogue(t, t, None, 0, None, False, None, None) is None
    assert n.matmul_epilogue(t, t, None, 0, None, True, None, t) is None
    assert n.matmul_epilogue(t, t.float(), None, 0, None, True, None, None) is None
    assert n.matmul_epilogue_backward(t, t, t, 2, None, None, True, True, True) is None
    assert n.newton_schulz(t, -1, 1.0, 1.0, 1.0, 1e-7, None) is None
    assert n.newton_schulz(t.half(), 5, 1.0, 1.0, 1.0, 1e-7, None) is None


def test_a_library_error_is_raised_by_either(gpu):
    import torch

    import kernel_library as kl

    # An operand past 4 GiB is refused by the library, before a launch.
    lhs = torch.empty(1, 1, dtype=torch.bfloat16, device=gpu)
    wide = torch.empty(1, 2**31 - 8, dtype=torch.bfloat16, device=gpu)
    out = torch.empty(1, 2**31 - 8, dtype=torch.bfloat16, device=gpu)
    kl.layer_norm(lhs)
    for _ in range(2):
        with pytest.raises(kl.epilogue._lib.KernelLibraryError, match="rc=5"):
            kl.matmul_epilogue(lhs, wide, out=out)


def test_sizes_past_32_bits_are_refused(gpu):
    """A size that a C int cannot hold is refused, not cut to the one it would become."""
    import torch

    import kernel_library as kl

    big = 2**32 + 8
    bf = dict(dtype=torch.bfloat16, device=gpu)
    none, eight = torch.empty(0, big, **bf), torch.zeros(8, 0, **bf)
    stats = torch.empty(0, device=gpu)
    for call in (lambda: kl.layer_norm(none), lambda: kl.layer_norm_backward(none, none, stats, stats),
                 lambda: kl.matmul_epilogue(none, none, rhs_transposed=True),
                 lambda: kl.matmul_epilogue(torch.empty(big, 0, **bf), eight, rhs_transposed=True),
                 lambda: kl.matmul_epilogue_backward(torch.empty(0, 0, **bf), none, none, rhs_transposed=True),
                 lambda: kl.newton_schulz(none), lambda: kl.newton_schulz(none.reshape(big, 0, 1)),
                 lambda: kl.newton_schulz(torch.zeros(4, 4, **bf), steps=2**32)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def test_negated_views_are_refused(gpu):
    import torch

    import kernel_library as kl

    v = torch.randn(8, 1, dtype=torch.complex64, device=gpu).conj().imag
    assert v.is_neg()
    with pytest.raises(ValueError, match="negated"):
        kl.layer_norm(v)


def test_two_threads_at_once(gpu):
    """Calls from two threads, each on a stream of its own: workspaces, errors and answers stay apart."""
    import threading

    import torch

    import kernel_library as kl

    bf = torch.bfloat16
    failed = []

    def work(seed):
        try:
            g = torch.Generator().manual_seed(seed)
            M, N, K = (40, 520, 2048) if seed else (70, 131, 333)
            lhs, rhs, r = (torch.randn(*s, generator=g).to(bf).to(gpu) for s in ((M, K), (K, N), (M, N)))
            grad = torch.randn(100 + seed, 2100, generator=g).to(bf).to(gpu)
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                def step():
                    y, mean, rstd = kl.layer_norm(r, stats=True)
                    out = kl.matmul_epilogue(lhs, rhs, None, "silu", y)
                    return (out, *kl.matmul_epilogue_backward(r, lhs, rhs, "silu", out)[:2],
                            kl.layer_norm_backward(out, r, mean, rstd)[0], kl.newton_schulz(grad))

                want = step()
                for _ in range(20):
                    with pytest.raises(ValueError, match="contraction mismatch"):
                        kl.matmul_epilogue(lhs, rhs[1:])
                    got = step()
                    stream.synchronize()
                    assert all(bool((a == b).all()) for a, b in zip(got, want))
        except BaseException as e:  # noqa: BLE001 -- reported by the main thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not failed, failed
    assert not any(t.is_alive() for t in threads)
