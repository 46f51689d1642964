"""Backward calls of the residual stream without rows: the sums over them are zeros, and what the join reads has to be there
(refusals only, before any GPU call; the pointers are never followed)."""

import pytest

from decik_amd import _lib
from test_more_ops_abi import P, error, norm

EMPTY = dict(rows=0, x=None, residual=None, y=None, h=None, dx=None, grad_y=None, post_weight=P, post_dtype=2)


@pytest.mark.parametrize("sums", [dict(dpost_weight=P), dict(dgate=P), dict(dweight=P), dict(dweight=P, dpost_weight=P, dgate=P)])
def test_sums_of_no_rows_need_the_channel_gate(sums):
    d = norm(**EMPTY, **sums, gate_kind=1, gate=None)
    assert "null gate" in error(_lib.lib().dk_residual_norm_bwd(d, None, 0, None))


@pytest.mark.parametrize("kind", [1, 2, 3])
def test_no_rows_and_no_sums_need_no_gate(kind):
    d = norm(**EMPTY, gate_kind=kind, gate=None)
    assert _lib.lib().dk_residual_norm_bwd(d, None, 0, None) == 0 and _lib.lib().dk_residual_norm_fwd(d, None) == 0
