"""Seam weights made from a differentiated leaf (a cast, a slice, a scaled copy) beside the leaf itself.

Discovery has to see the gradient that such a tensor brings to its leaf: the
capture pass records seams of the leaf alone, so a leaf with both would lose
that term from its per-example gradients, norms and clipped sum.
"""

from __future__ import annotations

import pytest
import torch
from test_capture import _capture_per_example, _check, _engine

from opaque_amd import capture

DERIVED = {
    "scaled": lambda w: 0.5 * w,
    "cast": lambda w: w.float().to(w.dtype),
    "slice": lambda w: torch.cat([w[:5], w[5:]]),
    "transposed": lambda w: w.t(),
}


@pytest.fixture(autouse=True)
def in_64_bits():
    torch.set_default_dtype(torch.float64)
    yield
    torch.set_default_dtype(torch.float32)


def both(loss_fn, params, n=3, width=8, seed=0):
    x = torch.randn(n, 5, width, generator=torch.Generator().manual_seed(seed))
    ref = torch.func.vmap(torch.func.grad(loss_fn), in_dims=(None, 0))(params, x)
    disc, sess, got, paths = _capture_per_example(_engine(loss_fn, batch_argnums=(1,)), (params, x), n)
    _check(ref, got)
    return {paths[k][0] for k in disc.eligible}, sess


@pytest.mark.parametrize("made", DERIVED)
@pytest.mark.parametrize("first", [False, True])
def test_linear_weight_tied_to_a_derived_one(made, first):
    g = torch.Generator().manual_seed(1)
    params = {"w": torch.randn(8, 8, generator=g), "v": torch.randn(8, 8, generator=g)}

    def loss_fn(p, x):
        ws = [p["w"], DERIVED[made](p["w"])]
        a, b = reversed(ws) if first else ws
        return (capture.linear(capture.linear(torch.tanh(capture.linear(x, a)), p["v"]), b) ** 2).sum()

    eligible, _ = both(loss_fn, params)
    assert eligible == {"v"}  # the leaf with a use outside its seam goes materialised, the others stay


def test_derived_weight_alone_leaves_the_other_seams():
    g = torch.Generator().manual_seed(2)
    params = {"w": torch.randn(8, 8, generator=g), "v": torch.randn(8, 8, generator=g)}
    eligible, sess = both(lambda p, x: (capture.linear(capture.linear(x, 2 * p["w"]), p["v"]) ** 2).sum(), params)
    assert eligible == {"v"} and len(sess.sites) == 1


@pytest.mark.parametrize("which", ["A", "B", "W"])
def test_lora_seam_of_a_derived_factor(which):
    """A derived factor takes its partner off the seams with it; the leaf's own seam use is not the whole of its gradient."""
    g = torch.Generator().manual_seed(3)
    frozen = torch.randn(8, 8, generator=g)
    params = {"A": torch.randn(8, 2, generator=g), "B": torch.randn(2, 8, generator=g),
              "A2": torch.randn(8, 2, generator=g), "B2": torch.randn(2, 8, generator=g),
              "W": torch.randn(8, 8, generator=g)}

    def loss_fn(p, x):
        a, b, w = p["A"], p["B"], frozen
        h = capture.lora_linear(x, w, a, b, 0.5)
        a, b, w = (2 * a if which == "A" else p["A2"]), (2 * b if which == "B" else p["B2"]), \
            (2 * p["W"] if which == "W" else frozen)
        y = capture.lora_linear(h, w, a, b, 0.5)
        return (y**2).sum() + 0.0 * sum(t.sum() for t in (p["A2"], p["B2"], p["W"]))

    both(loss_fn, params)


def test_lora_factors_made_from_tensors_outside_the_tree_stay_seams():
    """A base weight or factor that needs a gradient but hangs on no differentiated leaf does not matter."""
    g = torch.Generator().manual_seed(4)
    base = torch.randn(8, 8, generator=g, requires_grad=True)
    other = torch.randn(8, 2, generator=g, requires_grad=True)
    params = {"B": torch.randn(2, 8, generator=g)}
    eligible, sess = both(lambda p, x: (capture.lora_linear(x, 0.5 * base, 0.5 * other, p["B"], 0.5) ** 2).sum(), params)
    assert eligible == {"B"} and len(sess.sites) == 1


@pytest.mark.parametrize("which", ["gate", "down"])
def test_moe_of_a_derived_weight(which):
    g = torch.Generator().manual_seed(5)
    E, H, inter = 3, 8, 4
    params = {"gate": torch.randn(E, 2 * inter, H, generator=g) / 3, "down": torch.randn(E, H, inter, generator=g) / 2}

    def loss_fn(p, x):
        idx = torch.arange(2).expand(x.shape[0], 2)
        wts = torch.full((x.shape[0], 2), 0.5)
        h = capture.moe(x, p["gate"], p["down"], idx, wts)
        gate, down = (2 * p["gate"] if which == "gate" else p["gate"]), (2 * p["down"] if which == "down" else p["down"])
        return (capture.moe(h, gate, down, idx, wts) ** 2).sum()

    eligible, _ = both(loss_fn, params)
    assert not eligible
