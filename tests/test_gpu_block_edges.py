"""The ends of the norm, routing and tree-norm operators' ranges, on both host paths.

Tolerances count roundings of half a step, 2^-24 of a value in float32 and 2^-53 in float64, as the operators' own tests
do; each is derived beside its use.
"""

from __future__ import annotations

import math

import pytest
import torch

from opaque_amd import _native as N
from opaque_amd import capture, vocabulary
from opaque_amd.clipping import clipped_grad
from opaque_amd.experts import Router, route
from opaque_amd.global_norm import clip_by_global_norm, global_norm
from opaque_amd.normalization import RMSNorm, rms_norm, rms_norm_quantized
from test_gpu_route import check, logits

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
U = 2.0**-24


@pytest.fixture(params=[True, False], ids=["helper", "functions"])
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(vocabulary, "_host_ready", [None])


# ---------------------------------------------------------------------------
# The root-mean-square norm
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("gains,rows,stream", [((1 << 23) + 5, 1, BF16), ((1 << 22) + 1, 2, F32)], ids=str)
def test_more_gains_than_a_launch_takes(path, gains, rows, stream):
    """What the forward pass takes the backward pass takes: pieces of the batch have the bits that they have alone."""
    g = torch.Generator(device=DEV).manual_seed(7)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, gy = normal(gains, rows, 8).to(BF16), normal(gains, rows, 8).to(BF16)
    r, gh = normal(gains, rows, 8).to(stream), normal(gains, rows, 8).to(stream)
    w = (1 + 0.3 * normal(gains, 8)).to(BF16)
    one = lambda x, r, w: rms_norm(x, w, residual=r)

    def step(at):
        ts = [t[at].detach().requires_grad_() for t in (x, r, w)]
        outs = torch.func.vmap(one)(*ts)
        return [*outs, *torch.autograd.grad(outs, ts, [gy[at], gh[at]])]

    whole = step(slice(None))
    for first in (0, gains - 1000, *(k * gains // parts - 500 for parts in (2, 3, 5) for k in range(1, parts))):
        for a, b in zip(whole, step(slice(first, first + 1000))):
            assert torch.equal(a[first:first + 1000], b)
    # Half a step of bfloat16 and the float32 roundings (48 steps of the terms' size) for the last piece.
    h = (x[-1000:].float() + r[-1000:].float()).to(stream).double()
    inv = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    terms = gy[-1000:].double() * h * inv
    want = terms.sum(1)
    assert ((whole[4][-1000:].double() - want).abs() <= want.abs() * 2.0**-8 + 48 * U * terms.abs().sum(1)).all()


@pytest.mark.parametrize("gains,rows,width", [(6, 300, 24), (6, 300, 1001), (6, 300, 4096), (100, 300, 40), (511, 260, 8),
                                              (2, 2050, 200), (3, 40, 8200), (2, 40, 16400), (1, 40, 32768),
                                              (2, 40, 32768)])
@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (F32, F32), (F16, F32)], ids=str)
def test_several_strips_of_several_gains(gains, rows, width, dtype, stream):
    """Gains whose rows go to more than one workgroup: each sum against float64, dx with the bits of its example alone.

    A gain's sum takes rows + 64 float32 additions at most, each half a step of 2^-24 of the terms' sizes (with the terms'
    own products and 1 / sqrt), then half a step of its type.
    """
    words = N.load().odp_rms_norm_grad_scratch(gains * rows, width, gains)
    assert words > 4 * gains * width and words % (4 * gains * width) == 0  # two strips a gain at least
    g = torch.Generator(device=DEV).manual_seed(width + gains)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    size = torch.exp(normal(gains, rows, 1))
    ts = [(size * normal(gains, rows, width)).to(dtype), (size * normal(gains, rows, width)).to(stream),
          (1 + 0.3 * normal(gains, width)).to(dtype)]
    ts = [t.requires_grad_() for t in ts]
    gy, gh = normal(gains, rows, width).to(dtype), normal(gains, rows, width).to(stream)
    one = lambda x, r, w: rms_norm(x, w, residual=r)
    outs = torch.func.vmap(one)(*ts)
    dx, dr, dw = torch.autograd.grad(outs, ts, [gy, gh])
    h = outs[1].detach().double()
    terms = gy.double() * h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    want = terms.sum(1)
    slack = (rows + 64) * U * terms.abs().sum(1) + want.abs() * torch.finfo(dtype).eps / 2 + 1e-30
    worst = ((dw.double() - want).abs() - slack).max().item()
    assert worst <= 0, worst
    for i in {0, gains // 2, gains - 1}:
        alone = [t[i].detach().requires_grad_() for t in ts]
        a, b, c = torch.autograd.grad(one(*alone), alone, [gy[i], gh[i]])
        assert torch.equal(a, dx[i]) and torch.equal(b, dr[i])
        assert ((c.double() - want[i]).abs() <= slack[i]).all()


@pytest.mark.parametrize("shape", [(0, 24), (0, 3, 24), (4, 0, 24), (0, 0, 24)], ids=str)
def test_an_empty_batch_of_examples(path, shape):
    """vmap over no examples, or over examples without rows, with a gain or bias of each: empty results, zero gradients."""
    b = shape[0]
    x, r = (torch.ones(shape, device=DEV, requires_grad=True) for _ in range(2))
    w = torch.ones(b, 24, device=DEV, requires_grad=True)
    y, h = torch.func.vmap(lambda x, r, w: rms_norm(x, w, residual=r))(x, r, w)
    assert y.shape == h.shape == shape
    for t, d in zip((x, r, w), torch.autograd.grad([y, h], [x, r, w], [torch.ones_like(y), torch.ones_like(h)])):
        assert d.shape == t.shape and not d.any()
    total = lambda w, x: rms_norm(x, w).sum()
    for each in (w.detach(), torch.ones(24, device=DEV)):
        d = torch.func.vmap(torch.func.grad(total), in_dims=(0 if each.dim() == 2 else None, 0))(each, x.detach())
        assert d.shape == (b, 24) and not d.any()
    if len(shape) == 3:
        rows = torch.func.vmap(torch.func.vmap(torch.func.grad(total), in_dims=(None, 0)))(w.detach(), x.detach())
        assert rows.shape == shape
        flat = torch.func.vmap(torch.func.vmap(rms_norm, in_dims=(0, None)))(x, w)
        assert flat.shape == shape
    bias = torch.zeros(b, 24, device=DEV)
    index, weights = torch.func.vmap(lambda z, b: route(z, 2, bias=b))(x, bias)
    assert index.shape == weights.shape == (*shape[:-1], 2)
    dz = torch.func.vmap(torch.func.grad(lambda z, b: route(z, 2, bias=b)[1].sum()))(x.detach(), bias)
    assert dz.shape == shape


# ---------------------------------------------------------------------------
# Routing
# ---------------------------------------------------------------------------

LOW = [-1e2, -1e3, -1e4, -1e5, -1e9, torch.finfo(F32).min]


def biases(e, which, low):
    """Biases of some steps, and the experts of ``which`` switched off by a low finite one."""
    b = (torch.randn(e, generator=torch.Generator().manual_seed(e)) * 3).round() / 20
    at = {"one": [e // 3], "some": list(range(1, e, 5)), "first": list(range(e // 4)), "few stay": list(range(3, e)),
          "all": list(range(e)), "one of four stays": [i for i in range(e // 2) if i % (e // 4)],
          "mixed": list(range(e // 2))}[which]
    b[at] = low
    if which == "mixed":  # by several amounts, some equal
        b[at] = torch.tensor([low, 2 * low if low > -1e30 else low, -100.0, -40.0])[torch.arange(len(at)) % 4]
    return b.to(DEV)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e", [8, 16, 60, 256, 300, 1024])
@pytest.mark.parametrize("which", ["one", "some", "first", "few stay", "all", "one of four stays", "mixed"])
def test_experts_switched_off_by_a_low_bias(scores, e, which):
    """The float64 keys' choice whatever is below it, also where it reaches among the low ones or a group has one of them
    in its sum."""
    for low in LOW:
        b = biases(e, which, low)
        for dtype, spread in ((F32, 2.0), (BF16, 0.02)):
            z = logits(200, e, dtype, spread=spread)
            check(z, min(e, 6), scores=scores, bias=b)
            for best in ("top2", "max"):
                for groups, top_groups in ((4, 2), (4, 1), (2, 1)):
                    check(z, min(6, e // groups * top_groups), scores=scores, bias=b, groups=groups, top_groups=top_groups,
                          group_best=best, renormalize=False)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("spread", [0.3, 3.0, 30.0, 3000.0])
def test_biases_far_apart(scores, spread):
    """Biases over many times the scores' range, equal ones among them, deep choices too."""
    for e, k in ((8, 7), (64, 40), (256, 8), (256, 64), (1000, 16)):
        b = (torch.randn(e, generator=torch.Generator().manual_seed(e + 1)) * 8).round() / 8 * spread
        for s in (0.01, 2.0):
            z = logits(150, e, spread=s)
            check(z, k, scores=scores, bias=b.to(DEV))
            for best in ("top2", "max"):
                check(z, min(k, e // 2), scores=scores, bias=b.to(DEV), groups=8, top_groups=4, group_best=best)


# ---------------------------------------------------------------------------
# The router
# ---------------------------------------------------------------------------


class Block(torch.nn.Module):
    """Norm, router and experts; with ``plain`` the norm and the router in elementary operations."""

    def __init__(self, dtype, plain=False):
        super().__init__()
        self.plain = plain
        self.norm = RMSNorm(32, dtype=dtype)
        self.router = Router(32, 8, 2, scores="sigmoid", balance=True, scale=1.5, dtype=dtype)
        self.up, self.down = (torch.nn.Parameter(torch.empty(s, dtype=dtype)) for s in ((8, 48, 32), (8, 32, 24)))

    def forward(self, x):
        if not self.plain:
            n = self.norm(x)
            index, w = self.router(n)
        else:
            f = x.float()
            n = (f / torch.sqrt(f.square().mean(-1, keepdim=True) + 1e-6) * self.norm.weight.float()).to(x.dtype)
            p = torch.sigmoid(capture.linear(n, self.router.weight).float())
            index = (p + self.router.balance).topk(2, -1).indices
            w = p.gather(-1, index)
            w = 1.5 * w / w.sum(-1, keepdim=True)
        return x + capture.moe(n, self.up, self.down, index, w.to(n.dtype))


@pytest.mark.parametrize("dtype,tol", [(F32, 1e-5), (BF16, 2e-2)], ids=str)
def test_a_router_under_clipped_grad(path, dtype, tol):
    """The module in a DP step, its weight a full-weight seam, its bias moved between steps: as with elementary operations
    (1e-5 and 2e-2, the tolerances of the engine's own tests; the choices are the same, as the norms' roundings are)."""
    g = torch.Generator().manual_seed(5)
    own, plain = Block(F32), Block(F32, plain=True)
    for p in own.parameters():
        p.data = torch.randn(p.shape, generator=g) / p.shape[-1] ** 0.5 + (1 if p.dim() == 1 else 0)
    plain.load_state_dict(own.state_dict())
    own, plain = own.to(DEV, dtype), plain.to(DEV, dtype)
    x = torch.randn(5, 12, 32, generator=g).to(dtype).to(DEV)
    y = torch.randn(5, 12, 32, generator=g).to(DEV)
    steps = {}
    for m in (own, plain):
        def loss(params, x, y):
            return ((torch.func.functional_call(m, params, (x,)).float() - y) ** 2).mean()

        fn, st = clipped_grad(loss, clipping_norm=0.05, normalize_by=5, batch_argnums=(1, 2), return_aux=True)
        steps[m] = []
        for k in range(2):
            m.router.balance.copy_(0.2 * k * torch.linspace(-1, 1, 8, device=DEV))
            (got, aux), st = fn(dict(m.named_parameters()), x, y, state=st)
            steps[m].append({**got.pytree, "norms": aux.grad_norms, "losses": aux.loss_values})
    for a, b in zip(steps[own], steps[plain]):
        assert a["router.weight"].any() and a["norm.weight"].any()
        for k, t in a.items():
            assert (t.double() - b[k].double()).norm() <= tol * b[k].double().norm(), k
    assert own.router.balance.dtype == F32
    chosen = [own.router(own.norm(x))[0]]
    own.router.balance.zero_()
    assert not torch.equal(chosen[0], own.router(own.norm(x))[0])  # the bias is what moves the choice


# ---------------------------------------------------------------------------
# The norm of a tree
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("size", [5, 100, 40000])
@pytest.mark.parametrize("power", [1019, 600, 481, 479, 0, -479, -481, -600, -1000])
def test_float64_leaves_whose_squares_leave_float64(path, size, power):
    """Finite trees have finite norms, of one workgroup and of many, one launch and several: entries near 2^power.

    The norm is that of the entries over 2^power times 2^power, both exact: n additions of float64, 2^-53 n at most, n
    below 2^18, so 2^-35; the factor and the product one step of 2^-53 each beside it.
    """
    g = torch.Generator(device=DEV).manual_seed(size)
    # 2^1019 times 40000 values below 0.05 and 140 empty leaves (two launches): a norm below 2^1024.
    base = [0.02 + 0.03 * torch.rand(size, generator=g, device=DEV, dtype=F64) for _ in range(3)]
    unit = math.sqrt(sum(float(t.square().sum()) for t in base))
    for empty in (0, 140):
        grads = {f"k{i}": t * 2.0**power for i, t in enumerate(base)}
        grads |= {f"e{i}": torch.empty(0, device=DEV) for i in range(empty)}
        assert all(bool(t.isfinite().all()) for t in grads.values())
        norm = global_norm(grads)
        assert norm.dtype == F64 and abs(math.ldexp(float(norm), -power) / unit - 1) < 2.0**-35
        for over in (0.5, 4.0):
            got, same = clip_by_global_norm(grads, float(norm) / over)
            assert torch.equal(same, norm)
            for i, t in enumerate(base):
                back = got[f"k{i}"] * 2.0**-power
                # (entries of 2^-1000 / 32 and above keep their 53 bits)
                assert ((back - t / max(over, 1.0)).abs() <= 2.0**-50 * t).all()


def test_float64_leaves_of_all_sizes_together(path):
    """Entries on both sides of float64's squares in one tree, beside leaves of other types; a true infinity stays one."""
    tiny = torch.full((30000,), 1e-170, device=DEV, dtype=F64)
    for big, want in ((1e200, 1e200 * 2**0.5), (2.0**480, 2.0**480 * 2**0.5), (1e3, math.hypot(1e3 * 2**0.5, 30.0))):
        t = {"t": tiny, "b": torch.tensor([big, -big], device=DEV, dtype=F64), "f": torch.full((9,), 10.0, device=DEV),
             "h": torch.zeros(5, device=DEV, dtype=BF16)}
        got, norm = clip_by_global_norm(t, want / 2)
        assert abs(float(norm) / want - 1) < 1e-14
        assert abs(float(got["b"][0]) / (big / 2) - 1) < 1e-14 and float(got["b"][1]) < 0
        assert torch.allclose(got["f"], torch.full_like(got["f"], 5.0), rtol=1e-6, atol=0)
    only = {"t": tiny, "z": torch.zeros(40000, device=DEV)}
    assert abs(float(global_norm(only)) / (1e-170 * 30000**0.5) - 1) < 1e-12
    for bad, seen in ((float("inf"), math.isinf), (float("nan"), math.isnan)):
        t = {"b": torch.tensor([1e200, bad, 1e-200], device=DEV, dtype=F64)}
        assert seen(float(global_norm(t)))
    # Beyond float64 itself: an infinite norm, which makes finite entries 0.
    got, norm = clip_by_global_norm({"b": torch.full((4,), 1.5e308, device=DEV, dtype=F64)}, 1.0)
    assert norm.isinf() and not got["b"].any()


def test_tangents_are_refused_where_there_is_no_derivative(path):
    """A dual tensor in is an error, not a result without its tangent; plain tensors beside the level are none."""
    x, r = torch.randn(4, 32, device=DEV), torch.randn(4, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    want = rms_norm_quantized(x, w, residual=r)[2], global_norm({"a": x})
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for args in ((dual(x), r, w), (x, dual(r), w), (x, r, dual(w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                rms_norm_quantized(args[0], args[2], residual=args[1])
        for call in (global_norm, lambda t: clip_by_global_norm(t, 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call({"a": x, "b": dual(r)})
        assert torch.equal(rms_norm_quantized(x, w, residual=r)[2], want[0]) and global_norm({"a": x}) == want[1]


def test_views_whose_memory_holds_the_negative(path):
    """The imaginary part of a conjugate is a view with a negative bit, dense where it is one element; torch._neg_view
    makes one of any shape."""
    x, r, gy = (torch.randn(6, 64, device=DEV) for _ in range(3))
    w, b = torch.randn(64, device=DEV), 0.1 * torch.randn(64, device=DEV)
    neg = lambda t: torch._neg_view(-t)
    assert neg(x).is_neg() and torch.equal(neg(x), x)

    def step(x, r, w, gy):
        ts = [t.detach().requires_grad_() for t in (x, r, w)]
        outs = rms_norm(ts[0], ts[2], residual=ts[1])
        return [*outs, *torch.autograd.grad(outs, ts, [gy, gy])]

    for a, c in zip(step(x, r, w, gy), step(neg(x), neg(r), neg(w), neg(gy))):
        assert torch.equal(a, c)
    for a, c in zip(rms_norm_quantized(x, w, residual=r), rms_norm_quantized(neg(x), neg(w), residual=neg(r))):
        assert torch.equal(a.float(), c.float())
    z, zn = x.clone().requires_grad_(), neg(x).requires_grad_()
    (i, u), (j, v) = route(z, 4, bias=b), route(zn, 4, bias=neg(b))
    assert torch.equal(i, j) and torch.equal(u, v)
    g = torch.randn_like(u)
    assert torch.equal(torch.autograd.grad(u, z, g)[0], torch.autograd.grad(v, zn, neg(g))[0])
    one = torch.tensor(1.0 - 3.0j, device=DEV).conj().imag
    assert one.is_neg() and float(one) == 3.0
    tree, same = {"a": x, "b": one.clone().resolve_neg()}, {"a": neg(x), "b": one}
    (p, m), (q, n) = clip_by_global_norm(tree, 1.0), clip_by_global_norm(same, 1.0)
    assert torch.equal(m, n) and all(torch.equal(p[k], q[k]) for k in p) and float(q["b"]) > 0


def test_batched_gradients():
    """is_grads_batched is refused by name; torch.func's jacrev gives the same rows."""
    x, w = torch.randn(3, 16, device=DEV), torch.randn(16, device=DEV)
    leaf = x.clone().requires_grad_()
    y, (_, p) = rms_norm(leaf, w), route(leaf, 4)
    for out in (y, p):
        with pytest.raises(RuntimeError, match="is_grads_batched"):
            torch.autograd.grad(out, leaf, torch.ones(2, *out.shape, device=DEV), is_grads_batched=True, retain_graph=True)
    rows = torch.func.jacrev(lambda t: rms_norm(t, w))(x[0])
    for k in range(16):
        one = x[:1].clone().requires_grad_()
        assert torch.equal(rows[k], torch.autograd.grad(rms_norm(one, w)[0, k], one)[0][0])
