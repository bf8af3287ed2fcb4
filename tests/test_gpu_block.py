"""A block's norms, its router and its experts in one DP step: clipped_grad, noise and the bound on the step."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from opaque_amd import capture
from opaque_amd.clipping import auto_clipped_grad, clipped_grad
from opaque_amd.experts import route
from opaque_amd.global_norm import clip_by_global_norm
from opaque_amd.noise import gaussian_noise
from opaque_amd.normalization import rms_norm
from opaque_amd.random import key
from opaque_amd.types import NoisedPytree

pytestmark = pytest.mark.gpu

DEV = "cuda"
B, T, D, E, K, I = 5, 12, 32, 8, 2, 24


def params(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g) / s[-1] ** 0.5
    p = {"mix": r(D, D), "gain1": 1 + 0.2 * torch.randn(D, generator=g), "gain2": 1 + 0.2 * torch.randn(D, generator=g),
         "router": r(E, D), "up": r(E, 2 * I, D), "down": r(E, D, I), "gain3": 1 + 0.2 * torch.randn(D, generator=g)}
    return {k: v.to(dtype).to(DEV) for k, v in p.items()}


def batch(dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn(B, 1, 1, generator=g))
    return (size * torch.randn(B, T, D, generator=g)).to(dtype).to(DEV), torch.randn(B, T, D, generator=g).to(DEV)


def own_norm(x, w, r=None):
    return rms_norm(x, w, residual=r)


def plain_norm(x, w, r=None):
    h = x if r is None else x + r
    f = h.float()
    y = (f / torch.sqrt(f.square().mean(-1, keepdim=True) + 1e-6) * w.float()).to(x.dtype)
    return y if r is None else (y, h)


def own_route(z, bias):
    return route(z, K, scores="sigmoid", bias=bias, groups=4, top_groups=2, scale=1.5)


def plain_route(z, bias):
    p = torch.sigmoid(z.float())
    with torch.no_grad():
        each = (p + bias).unflatten(-1, (4, 2))
        shut = torch.ones_like(each[..., 0]).scatter(-1, each.sum(-1).topk(2, -1).indices, 0.0).bool()
        index = (p + bias).masked_fill(shut.repeat_interleave(2, -1), -torch.inf).topk(K, -1).indices
    w = p.gather(-1, index)
    return index, 1.5 * w / w.sum(-1, keepdim=True)


def loss(norm, choose, bias):
    def f(p, x, y):
        h = capture.linear(norm(x, p["gain1"]), p["mix"])
        n, h = norm(h, p["gain2"], x)
        index, weights = choose(capture.linear(n, p["router"]), bias)
        out = capture.moe(n, p["up"], p["down"], index, weights.to(n.dtype))
        last, _ = norm(out, p["gain3"], h)
        return ((last.float() - y) ** 2).mean()

    return f


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("auto", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_dp_step(dtype, auto):
    """Norms and clipped sums as with the same model's elementary operations, gains and router among them.  float32: the
    tolerance the engine's own tests have (1e-5); bfloat16: 2e-2, theirs, where no token's choice hangs on a rounding."""
    p, (x, y) = params(dtype), batch(dtype)
    bias = 0.05 * torch.randn(E, generator=torch.Generator().manual_seed(3)).to(DEV)
    make = (lambda f: auto_clipped_grad(f, R=1.0, normalize_by=B, batch_argnums=(1, 2), return_aux=True)) if auto else (
        lambda f: clipped_grad(f, clipping_norm=0.05, normalize_by=B, batch_argnums=(1, 2), return_aux=True))
    fn, st = make(loss(own_norm, own_route, bias))
    (got, aux), _ = fn(p, x, y, state=st)
    fn, st = make(loss(plain_norm, plain_route, bias))
    (want, waux), _ = fn(p, x, y, state=st)
    tol = 1e-5 if dtype == torch.float32 else 2e-2
    assert rel(aux.grad_norms, waux.grad_norms) < tol and rel(aux.loss_values, waux.loss_values) < tol
    for k in p:
        assert got.pytree[k].dtype == dtype and rel(got.pytree[k], want.pytree[k]) < tol, k


def test_noise_and_the_bound_on_the_step():
    p, (x, y) = params(torch.bfloat16), batch(torch.bfloat16)
    bias = torch.zeros(E, device=DEV)
    fn, st = auto_clipped_grad(loss(own_norm, own_route, bias), R=1.0, normalize_by=B, batch_argnums=(1, 2))
    grads, st = fn(p, x, y, state=st)
    noise, ns = gaussian_noise(noise_multiplier=0.5, key=key(1))
    noisy, ns = noise(grads, ns)
    assert isinstance(noisy, NoisedPytree)
    total = sum(float(t.double().square().sum()) for t in noisy.pytree.values()) ** 0.5
    step, norm = clip_by_global_norm(noisy, 0.1)
    assert abs(float(norm) - total) < 1e-6 * total and total > 0.1
    size = sum(float(t.double().square().sum()) for t in step.values()) ** 0.5
    assert abs(size - 0.1) < 0.1 * 2.0**-8 and set(step) == set(p)
    p = {k: t - step[k] for k, t in p.items()}
    again, _ = fn(p, x, y, state=st)  # the plan is kept from the first call
    assert all(t.isfinite().all() for t in again.pytree.values())


def test_microbatches_agree():
    """The step in pieces gives the step."""
    p, (x, y) = params(torch.float32), batch(torch.float32)
    f = loss(own_norm, own_route, torch.zeros(E, device=DEV))
    whole, st = clipped_grad(f, clipping_norm=0.05, normalize_by=B, batch_argnums=(1, 2))
    a, _ = whole(p, x, y, state=st)
    parts, st = clipped_grad(f, clipping_norm=0.05, normalize_by=B, batch_argnums=(1, 2), microbatch_size=2)
    b, _ = parts(p, x, y, state=st)
    for k in p:
        assert rel(a.pytree[k], b.pytree[k]) < 1e-5


def test_a_block_without_dp():
    """The block under plain autograd, in a graph: forward, gradients and the bounded step replayed on new inputs."""
    p, (x, y) = params(torch.float32), batch(torch.float32)
    leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
    f = loss(own_norm, own_route, torch.zeros(E, device=DEV))

    def step():
        grads = torch.autograd.grad(f(leaves, x, y), list(leaves.values()))
        return clip_by_global_norm(dict(zip(leaves, grads)), 0.01)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, norm = step()
    for k in range(3):
        nx, ny = batch(torch.float32, seed=k)
        x.copy_(nx), y.copy_(ny)
        graph.replay()
        torch.cuda.synchronize()
        want, wnorm = step()
        assert abs(float(norm) / float(wnorm) - 1) < 1e-5
        for key_ in leaves:
            assert rel(out[key_], want[key_]) < 1e-5


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2e-2)])
def test_a_model_on_its_own_norms(dtype, tol):
    """A Hugging Face Llama whose norm gains train under clipped_grad, with its norms replaced and without."""
    transformers = pytest.importorskip("transformers")
    from opaque_amd.normalization import RMSNorm, route_norms

    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(vocab_size=128, hidden_size=64, intermediate_size=96, num_hidden_layers=2,
                                   num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=128,
                                   attn_implementation="eager")
    m = transformers.LlamaForCausalLM(cfg).eval().to(dtype).to(DEV)
    for p in m.parameters():
        p.requires_grad_(False)
    gains = {k: p.requires_grad_() for k, p in m.named_parameters() if "norm" in k}
    assert len(gains) == 5
    g = torch.Generator().manual_seed(1)
    ids, labels = (torch.randint(0, 128, (6, 24), generator=g).to(DEV) for _ in range(2))

    def loss_fn(params, ids, labels):
        fixed = {k: v for k, v in m.named_parameters() if k not in params}
        return torch.func.functional_call(m, {**fixed, **params}, (ids.unsqueeze(0),),
                                          {"labels": labels.unsqueeze(0)}).loss

    def step():
        fn, st = auto_clipped_grad(loss_fn, R=1.0, normalize_by=6, batch_argnums=(1, 2), return_aux=True)
        (grads, aux), _ = fn(gains, ids, labels, state=st)
        return grads.pytree, aux

    want, waux = step()
    kind = type(m.model.norm)
    assert len(route_norms(m, (kind,))) == 5 and type(m.model.norm) is RMSNorm
    got, aux = step()
    assert rel(aux.grad_norms, waux.grad_norms) < tol and rel(aux.loss_values, waux.loss_values) < tol
    for k in gains:
        assert rel(got[k], want[k]) < tol, k
