"""Seams under a vmap of the loss's own, inside the engine's (no kernel runs)."""

from __future__ import annotations

import pytest
import torch
from test_capture import _capture_per_example, _check, _engine

from opaque_amd import capture


@pytest.fixture(autouse=True)
def in_64_bits():
    torch.set_default_dtype(torch.float64)
    yield
    torch.set_default_dtype(torch.float32)


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


FROZEN = rand(8, 8, seed=5)
IDX, WTS = torch.tensor([0, 2]), torch.tensor([0.25, 0.75], dtype=torch.float64)
CASES = {
    "linear": ({"w": rand(8, 8, seed=1), "b": rand(8, seed=2)}, 1,
               lambda p: lambda r: capture.linear(r, p["w"], p["b"])),
    "lora": ({"A": rand(8, 2, seed=3), "B": rand(2, 8, seed=4), "b": rand(8, seed=2)}, 1,
             lambda p: lambda r: capture.lora_linear(r, FROZEN, p["A"], p["B"], 0.5, p["b"])),
    "moe": ({"gate": rand(3, 8, 8, seed=6), "down": rand(3, 8, 4, seed=7)}, 6,
            lambda p: lambda r: capture.moe(r, p["gate"], p["down"], IDX, WTS)),
}


@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("case", CASES)
def test_a_seam_under_an_inner_vmap_is_recorded_once(case, dim):
    params, sites, make = CASES[case]

    def loss(p, x):
        return torch.func.vmap(make(p), in_dims=dim)(x if dim == 0 else x.t()).sin().sum()

    x = rand(3, 5, 8, seed=9)
    ref = torch.func.vmap(torch.func.grad(loss), in_dims=(None, 0))(params, x)
    disc, sess, got, paths = _capture_per_example(_engine(loss, batch_argnums=(1,)), (params, x), 3)
    _check(ref, got)
    assert len(sess.sites) == sites and {paths[k][0] for k in disc.eligible} == set(params) - {"b"}
