"""Scalars of the vocabulary operators that float32 does not hold are refused (no GPU: every call returns before device work)."""

from __future__ import annotations

import math

import pytest
import torch

from opaque_amd import _native as N
from opaque_amd import vocabulary

BAD = 64  # a non-null, aligned address; never read


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from opaque_amd import build

        build.build()
    return N.load()


@pytest.mark.parametrize("cap", [-1.0, math.inf, math.nan, 1e-40])
def test_softcaps_at_the_entry_points(lib, cap):
    rc = lib.odp_xent_losses(None, N.DTYPE_BF16, BAD, 0, 8, BAD, BAD, BAD, BAD, 8, 10, cap, BAD, BAD, BAD, None, 0)
    assert rc == N.ERR_INVALID_ARGUMENT and "softcap" in N.last_error()
    rc = lib.odp_xent_dlogits(None, N.DTYPE_BF16, BAD, 0, 8, BAD, BAD, BAD, BAD, 8, 600, cap, 0, 10, BAD, BAD, 1, None,
                              None, 0, BAD, 256, BAD)
    assert rc == N.ERR_INVALID_ARGUMENT and "softcap" in N.last_error()


@pytest.mark.parametrize("scale", [math.inf, math.nan])
def test_scales_at_the_entry_points(lib, scale):
    for rc in (lib.odp_embed_rows(None, N.DTYPE_F32, BAD, 8, 0, BAD, 8, 10, 8, scale, BAD),
               lib.odp_embed_grad(None, N.DTYPE_F32, BAD, 8, 0, 8, BAD, BAD, 10, scale, BAD, BAD),
               lib.odp_embed_sqnorm(None, N.DTYPE_F32, BAD, 8, 0, 8, BAD, BAD, BAD, 10, scale, BAD, BAD, BAD, BAD, BAD, 4,
                                    0, BAD),
               lib.odp_embed_clipped_sum(None, N.DTYPE_F32, BAD, 8, 0, 8, BAD, BAD, BAD, 10, scale, BAD, BAD, BAD, BAD,
                                         1.0, N.DTYPE_F32, BAD, None)):
        assert rc == N.ERR_INVALID_ARGUMENT and "scale" in N.last_error()


@pytest.mark.gpu
def test_scalars_outside_float32_are_refused():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(9, 16, device="cuda")
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    for cap in (1e39, 1e-39, 0.0, math.nan):
        with pytest.raises(ValueError):
            vocabulary.linear_cross_entropy(x, w, y, softcap=cap)
    for scale in (1e39, -1e39, math.nan):
        with pytest.raises(ValueError):
            vocabulary.embedding(y, w, scale=scale)
