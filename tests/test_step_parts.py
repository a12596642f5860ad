"""What mi_residual_norm_backward plans for where outputs are left out (no call here touches a GPU)."""

from __future__ import annotations

import pytest

from kernel_library import _lib
from test_step_refusals import _need, _rn_bwd


@pytest.mark.parametrize("D", [64, 9000])
def test_sums_by_gate_are_those_of_the_gate(D):
    """post_weight's gradient alone takes the partial sums that it takes beside the gate's: rows of one gate each."""
    query, size = _lib.lib().mi_residual_norm_backward_workspace, dict(rows=2048, gates=1024, D=D, ldx=D, lddy=D)
    alone = _need(query, _rn_bwd(dweight=None, dgate=None, **size))
    assert alone == _need(query, _rn_bwd(dweight=None, **size)) == _need(query, _rn_bwd(dweight=None, dpost_weight=None, **size))
    assert alone >= 1024 * D * 4
    # dweight alone needs none of it, a gate for each row no sums by gate.
    assert _need(query, _rn_bwd(dgate=None, dpost_weight=None, **size)) < alone
    assert _need(query, _rn_bwd(dweight=None, dgate=None, **(size | dict(gates=2048)))) < alone
