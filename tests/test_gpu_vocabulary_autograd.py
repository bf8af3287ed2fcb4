"""The vocabulary operators as autograd nodes: what they refuse, what they hold, which gradients they give."""

from __future__ import annotations

import math

import pytest
import torch
import torch.utils.checkpoint

from opaque_amd import vocabulary
from opaque_amd.vocabulary import embedding, linear_cross_entropy

pytestmark = pytest.mark.gpu

DEV = "cuda"


def inputs(n=8, width=16, vocab=30, dtype=torch.float32, seed=5):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(n, width, generator=g), torch.randn(vocab, width, generator=g) / math.sqrt(width)
    return x.to(dtype).to(DEV), w.to(dtype).to(DEV), torch.randint(0, vocab, (n,), generator=g).to(DEV)


@pytest.fixture(params=[True, False], ids=["helper", "functions"])
def route(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(vocabulary, "_host_ready", [None])


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("trained", ["x", "w", "xw"])
def test_a_second_derivative_of_the_loss_is_an_error(route, reduction, trained):
    """Also where the gradient that comes in is a constant: the first derivative depends on x and the head."""
    x, w, y = inputs()
    x.requires_grad_("x" in trained), w.requires_grad_("w" in trained)
    wanted = [t for t in (x, w) if t.requires_grad]
    loss = linear_cross_entropy(x, w, y, reduction=reduction)
    gl = torch.ones_like(loss)
    first = torch.autograd.grad(loss, wanted, gl, create_graph=True)
    plain = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction), wanted, gl)
    for d, p in zip(first, plain):
        assert d.requires_grad and torch.equal(d.detach(), p) and not p.requires_grad
        for t in wanted:
            with pytest.raises(RuntimeError):
                torch.autograd.grad(d.square().sum(), t, retain_graph=True)
    loss = linear_cross_entropy(x, w, y, reduction=reduction).sum()
    first = torch.autograd.grad(loss, wanted, create_graph=True)
    with pytest.raises(RuntimeError):
        (loss + sum(d.square().sum() for d in first)).backward()


def test_first_derivatives_under_create_graph_are_usable(route):
    """backward(create_graph=True) itself is no second derivative; a penalty on other tensors differentiates."""
    x, w, y = inputs()
    x.requires_grad_(), w.requires_grad_()
    linear_cross_entropy(x, w, y).backward(create_graph=True)
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    scale = torch.tensor(2.0, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(linear_cross_entropy(x, w, y), [x], create_graph=True)
    (ds,) = torch.autograd.grad((scale * dx).square().sum(), [scale])
    assert torch.allclose(ds, 2 * scale.detach() * dx.detach().square().sum())


def test_a_second_derivative_of_the_lookup(route):
    """The table's gradient is linear in the gradient that comes in, which the kernels do not differentiate; it does
    not depend on the table."""
    _, w, y = inputs()
    w.requires_grad_()
    go = torch.ones(y.numel(), w.shape[1], device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(embedding(y, w), [w], go, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dw.sum(), [go])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("kept", [True, False])
def test_a_head_that_trains_where_x_does_not(route, dtype, kept, monkeypatch):
    """Each gradient alone has the bits that both together have."""
    if not kept:
        monkeypatch.setattr(vocabulary, "KEEP_BYTES", 0)
    x, w, y = inputs(60, 136, 700, dtype)
    both = torch.autograd.grad(linear_cross_entropy(x.requires_grad_(), w.requires_grad_(), y), [x, w])
    (dw,) = torch.autograd.grad(linear_cross_entropy(x.detach(), w, y), [w])
    (dx,) = torch.autograd.grad(linear_cross_entropy(x, w.detach(), y), [x])
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])


@pytest.mark.parametrize("trained", ["x", "xw"])
def test_saved_tensors_go_through_autograds_hooks(trained):
    """What the backward needs is offered to saved-tensor hooks (offloading), rows and head among it, and comes back
    from them."""
    x, w, y = inputs(60, 136, 700)
    x.requires_grad_(), w.requires_grad_("w" in trained)
    wanted = [t for t in (x, w) if t.requires_grad]
    want = torch.autograd.grad(linear_cross_entropy(x, w, y), wanted)
    packed = []

    def pack(t):
        packed.append(tuple(t.shape))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        loss = linear_cross_entropy(x, w, y)
    assert packed.count((60, 136)) == packed.count((700, 136)) == 1
    for a, b in zip(torch.autograd.grad(loss, wanted), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("use_reentrant", [True, False])
def test_under_checkpointing(use_reentrant):
    x, w, y = inputs(60, 136, 700)
    x.requires_grad_(), w.requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(torch.tanh(x), w, y), [x, w])
    loss = torch.utils.checkpoint.checkpoint(lambda a, b: linear_cross_entropy(torch.tanh(a), b, y), x, w,
                                             use_reentrant=use_reentrant)
    loss.backward()
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])


def test_nothing_is_held_after_the_backward():
    """The packed rows go with the kept logits when the backward is through, while the loss itself is still held."""
    n, width, vocab = 2048, 1024, 4096
    x, w, y = inputs(n, width, vocab, torch.bfloat16)
    x.requires_grad_()

    def held():
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = linear_cross_entropy(x, w, y)
        mid = torch.cuda.memory_allocated() - before
        loss.backward()
        x.grad = None
        return mid, torch.cuda.memory_allocated() - before, loss

    held()
    mid, after, loss = held()
    assert mid >= 4 * n * vocab + 2 * n * width and after < 2 * n * width // 4


def test_a_checkpointed_loss_holds_nothing():
    """Non-reentrant checkpointing drops what the forward saved, the packed rows too."""
    n, width, vocab = 2048, 1024, 4096
    x, w, y = inputs(n, width, vocab, torch.bfloat16)
    x.requires_grad_()

    def held():
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = torch.utils.checkpoint.checkpoint(lambda a: linear_cross_entropy(a, w, y), x, use_reentrant=False)
        return torch.cuda.memory_allocated() - before, loss

    held()
    mid, loss = held()
    assert mid < 2 * n * width // 4


@pytest.mark.parametrize("pitch", [(1 << 20) - 8, 1 << 20, (1 << 20) + 3])
def test_heads_of_far_apart_rows(route, pitch):
    """Rows of the head farther apart than the kernels' offsets reach are copied, not refused."""
    x, w, y = inputs(20, 64, 3)
    far = torch.zeros(3, pitch, device=DEV)
    far[:, :64] = w
    v = far[:, :64].requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(x.requires_grad_(), w.requires_grad_(), y), [x, w])
    for a, b in zip(torch.autograd.grad(linear_cross_entropy(x, v, y), [x, v]), want):
        assert torch.equal(a, b)


def test_kept_logits_of_all_live_losses_are_bounded(monkeypatch):
    """Losses that wait for their backward passes share KEEP_BYTES; what one gives back the next may keep."""
    n, width, vocab = 512, 1024, 4096
    logits = 4 * n * vocab
    x, w, y = inputs(n, width, vocab, torch.bfloat16)
    x.requires_grad_()
    monkeypatch.setattr(vocabulary, "KEEP_BYTES", 2 * logits + 1)

    def growth():
        before = torch.cuda.memory_allocated()
        loss = linear_cross_entropy(x, w, y)
        return loss, torch.cuda.memory_allocated() - before >= logits

    torch.autograd.grad(growth()[0], [x])
    live = [growth() for _ in range(3)]
    assert [kept for _, kept in live] == [True, True, False]
    grads = [torch.autograd.grad(live[0][0], [x])[0]]
    again = growth()
    assert again[1]
    grads += [torch.autograd.grad(loss, [x])[0] for loss, _ in (live[1], live[2], again)]
    for g in grads[1:]:
        assert torch.equal(g, grads[0])
    del live, again, growth


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_an_error(route, requires_grad):
    """A tangent on x, the head or the table is refused, not dropped."""
    x, w, y = inputs()
    with torch.autograd.forward_ad.dual_level():
        dual = [torch.autograd.forward_ad.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t))
                for t in (x, w)]
        for call in (lambda: linear_cross_entropy(dual[0], w, y), lambda: linear_cross_entropy(x, dual[1], y),
                     lambda: embedding(y, dual[1])):
            with pytest.raises(RuntimeError):
                call()
    for f, t in ((lambda a: linear_cross_entropy(a, w, y), x), (lambda a: embedding(y, a), w)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))


def test_in_inference_mode(route):
    x, w, y = inputs()
    want = linear_cross_entropy(x, w, y), embedding(y, w)
    with torch.inference_mode():
        got = linear_cross_entropy(x.clone(), w.clone(), y.clone()), embedding(y.clone(), w.clone())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("back", ["cpu", "half"])
def test_saved_tensors_that_come_back_otherwise_are_refused(route, back):
    """Hooks that leave a saved tensor on the host, or in another type, give an error: the kernels take addresses."""
    x, w, y = inputs(60, 136, 700)
    x.requires_grad_(), w.requires_grad_()
    change = {"cpu": lambda t: t.cpu(), "half": lambda t: t.to(torch.float64) if t.is_floating_point() else t}[back]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        loss, rows = linear_cross_entropy(x, w, y), embedding(y, w)
    with pytest.raises((RuntimeError, TypeError)):
        torch.autograd.grad(loss, [x, w])
    if back == "cpu":
        with pytest.raises(RuntimeError):
            torch.autograd.grad(rows, [w], torch.ones_like(rows))


def test_saved_heads_come_back_in_another_layout(route):
    """A hook may change strides: transposed heads and rows give the same bits."""
    x, w, y = inputs(60, 136, 700)
    x.requires_grad_(), w.requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(x, w, y), [x, w])
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turned):
        loss = linear_cross_entropy(x, w, y)
    for a, b in zip(torch.autograd.grad(loss, [x, w]), want):
        assert torch.equal(a, b)
