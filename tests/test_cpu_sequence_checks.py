"""More of what the host side of the sequence-policy operators refuses (nothing is launched)."""
import math

import pytest

from test_cpu_sequence_ops import call, filled


@pytest.mark.parametrize("bad", [math.inf, 3e38, 1e19, 1e-19, 1e-45])
def test_distill_refuses_temperatures_without_a_square_or_reciprocal(bad):
    """At an infinite temperature every absent action (-inf times 0) made the row NaN."""
    from xuance_amd import _lib
    ok = dict(N=4, A=16, K=4, temperature=1.0, grad_scale=1.0, ld=16, ld_d=16)
    assert call("xrl_distill_loss", filled(_lib.Distill, **{**ok, "temperature": bad})) == -1
    assert b"temperature" in _lib.load().xrl_last_error()
