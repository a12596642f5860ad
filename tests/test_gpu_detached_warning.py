"""A forward operator says so where autograd is recording and its result will not be recorded."""

import warnings

import pytest

pytestmark = pytest.mark.gpu


def _calls(gpu):
    """(operator, call with its operand t), t in every place a gradient could come from."""
    import torch

    import kernel_library as kl

    def bf(*shape):
        return torch.randn(*shape, device=gpu).bfloat16()

    x, w, lhs, rhs, b, r = bf(8, 64), bf(64), bf(8, 64), bf(64, 32), bf(32), bf(8, 32)
    wide = bf(8, 80)[:, :64]  # left to the Python body
    return [(kl.layer_norm, x, lambda t: kl.layer_norm(t, w)), (kl.layer_norm, w, lambda t: kl.layer_norm(x, t, w)),
            (kl.layer_norm, w, lambda t: kl.layer_norm(x, w, t)), (kl.layer_norm, w, lambda t: kl.layer_norm(wide, t)),
            (kl.matmul_epilogue, lhs, lambda t: kl.matmul_epilogue(t, rhs)),
            (kl.matmul_epilogue, rhs, lambda t: kl.matmul_epilogue(lhs, t)),
            (kl.matmul_epilogue, b, lambda t: kl.matmul_epilogue(lhs, rhs, t)),
            (kl.matmul_epilogue, r, lambda t: kl.matmul_epilogue(lhs, rhs, residual=t)),
            (kl.matmul_epilogue, rhs, lambda t: kl.matmul_epilogue(lhs, t, cfg=kl.epilogue_configs()[0])),
            (kl.newton_schulz, lhs, lambda t: kl.newton_schulz(t))]


def test_warns_where_a_gradient_is_lost(gpu):
    import torch

    for op, t, call in _calls(gpu):
        for _ in range(2):  # the second by the native call, where it takes it
            with warnings.catch_warnings():
                warnings.simplefilter("error")
                want = call(t)
            with pytest.warns(UserWarning, match=f"{op.__name__} records nothing for autograd") as seen:
                got = call(t.clone().requires_grad_())
            assert len(seen) == 1 and seen[0].filename == __file__
            assert not got.requires_grad and torch.equal(got, want)


def test_quiet_where_none_is_expected(gpu):
    import torch

    class Own(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t, call):
            return call(t)

    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for _, t, call in _calls(gpu):
            call(t)
            t = t.clone().requires_grad_()
            with torch.no_grad():
                call(t)
            assert Own.apply(t, call).requires_grad


def test_a_warning_made_an_error_is_raised(gpu):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for op, t, call in _calls(gpu):
            with pytest.raises(UserWarning, match=op.__name__):
                call(t.clone().requires_grad_())
