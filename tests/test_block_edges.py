"""The ends of the norm, routing and tree-norm operators' ranges that need no GPU."""

from __future__ import annotations

from opaque_amd import _native as N
from opaque_amd import normalization


def test_gains_of_a_gradient_call_match_the_header():
    text = (N.LIB_PATH.parents[1] / "include" / "opaque_dp.h").read_text()
    assert "ODP_NORM_GRAD_GAINS ((int64_t)1 << 21)" in text and normalization._GRAD_GAINS == 1 << 21
