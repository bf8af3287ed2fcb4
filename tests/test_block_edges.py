"""The ends of the norm, routing and tree-norm operators' ranges that need no GPU."""

from __future__ import annotations

import pytest

from opaque_amd import _native as N
from opaque_amd import normalization

F32, BF16 = N.DTYPE_F32, N.DTYPE_BF16
BAD = 64  # a non-null, aligned address; never read


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from opaque_amd import build

        build.build()
    return N.load()


def test_an_empty_batch_has_no_gains_and_no_biases(lib):
    norm = lambda n, gains: lib.odp_rms_norm(None, BF16, BF16, BF16, BAD, 8, None, 0, n, 8, BAD, 8, gains, 1e-6, 0.0, 0,
                                             BAD, None, None, None)
    grad = lambda n, gains: lib.odp_rms_norm_grad(None, BF16, BF16, BF16, BAD, 8, BAD, BAD, 8, None, 0, n, 8, BAD, 8, gains,
                                                  0.0, BAD, BAD, None, BAD)
    route = lambda n, biases: lib.odp_route(None, F32, BAD, 8, n, 8, 0, BAD, biases, 1, 1, 0, 2, 1, 1.0, BAD, BAD)
    for call, text in ((norm, "do not divide into"), (grad, "do not divide into"), (route, "do not divide into")):
        assert call(0, 0) == call(0, 3) == N.ODP_OK, N.last_error()
        for n, count in ((4, 0), (4, 3), (0, -1), (4, -2)):
            assert call(n, count) == N.ERR_INVALID_ARGUMENT and text in N.last_error()


def test_gains_of_a_gradient_call_match_the_header():
    text = (N.LIB_PATH.parents[1] / "include" / "opaque_dp.h").read_text()
    assert "ODP_NORM_GRAD_GAINS ((int64_t)1 << 21)" in text and normalization._GRAD_GAINS == 1 << 21
