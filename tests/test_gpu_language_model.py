"""The example that trains a language model with its vocabulary ends under DP-SGD."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "dp_language_model.py")


def load():
    spec = importlib.util.spec_from_file_location("dp_language_model", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_example_trains():
    losses = load().train(vocab=512, width=128, blocks=1, examples=8, seq=32, steps=12, noise=0.0, report=lambda _: None)
    assert all(torch.isfinite(torch.tensor(losses))) and sum(losses[-4:]) < sum(losses[:4])


def test_every_weight_is_a_seam():
    """No leaf falls to a dense per-example gradient."""
    m = load()
    params = m.init(512, 128, 1, seed=0)
    tokens, target = m.batch(4, 16, torch.arange(512).roll(1), seed=0)
    grad_fn, state = m.auto_clipped_grad(m.loss_fn, R=1.0, normalize_by=4.0, batch_argnums=(1, 2))
    got, state = grad_fn(params, tokens, target, state=state)
    plan = grad_fn.engine._plan
    assert len(plan._embeds) == 1 and "sqnorm" not in {i[0] for i in plan.launch_info}
    assert sum(1 for k in plan._ext_keys if k[0] == "linx") == len(params) - 1
    # The reference's way: dense per-example gradients, AUTO-S, sum.
    per = torch.func.vmap(torch.func.grad(m.loss_fn), in_dims=(None, 0, 0))(params, tokens, target)
    norms = sum(g.double().flatten(1).square().sum(1) for g in per.values()).sqrt()
    for k, g in per.items():
        want = (g.double() / (norms + 0.01).view(-1, *[1] * (g.dim() - 1))).sum(0) / 4.0
        assert float((got.pytree[k].double() - want).norm() / want.norm()) < 2e-2
