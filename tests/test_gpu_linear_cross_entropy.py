"""linear_cross_entropy: losses and gradients against float64.

The bounds follow the computation.  A logit u is a float32 sum of D products:
|du| <= 2 D 2^-24 sum|x w| =: Z (the 2 covers whichever way the matrix cores
round their partial sums).  exp(z - lse) is off by a relative Z, the row's
largest Z (from lse) and (8 + |z - lse|) 2^-22 (the exponential's argument and
its last place).  d is that times g, rounded to the inputs' type (u); dx and
dW add V and N such terms in float32 and round once.
"""

from __future__ import annotations

import math

import pytest
import torch

from opaque_amd import vocabulary
from opaque_amd.clipping import clipped_grad
from opaque_amd.vocabulary import Embedding, embedding, linear_cross_entropy
from oracle import dp_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0**-24
HALF_ULP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
LEAST = 2.0**-120
DTYPES = [torch.float32, torch.bfloat16]


def inputs(n, width, vocab, dtype, seed=0, size=1.0, ignored=0.25):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(vocab, width, generator=g) / math.sqrt(width)).to(dtype)
    y = torch.randint(0, vocab, (n,), generator=g)
    lean = torch.rand(n, 1, generator=g) * 1.5 * math.log(vocab)
    x = (size * (torch.randn(n, width, generator=g) + lean * w[y].float())).to(dtype)
    y[torch.rand(n, generator=g) < ignored] = -100
    gl = torch.randn(n, generator=g)
    return x, w, y, gl


def reference(x, w, y, gl, softcap, dtype):
    """float64 (losses, dx, dW) and their bounds."""
    x, w, gl = x.double().to(DEV), w.double().to(DEV), gl.double().to(DEV)
    y = y.to(DEV)
    n, vocab, width = x.shape[0], w.shape[0], x.shape[1]
    live = y != -100
    u = x @ w.t()
    Z = 2 * width * U32 * (x.abs() @ w.abs().t())
    c = softcap or 0.0
    z = c * torch.tanh(u / c) if c else u
    Z = Z + (c * 2.0**-21 if c else 0.0)
    lse = torch.logsumexp(z, 1, keepdim=True)
    r = Z + Z.max(1, keepdim=True).values + (8 + (z - lse).abs()) * 2.0**-22
    at = torch.where(live, y, 0)
    zt = z.gather(1, at.unsqueeze(1)).squeeze(1)
    losses = torch.where(live, lse.squeeze(1) - zt, 0.0)
    lb = torch.where(live, 2 * Z.max(1).values + (16 + (zt - lse.squeeze(1)).abs()) * 2.0**-22
                     + 4 * U32 * (lse.squeeze(1).abs() + zt.abs()), 0.0)
    p = torch.exp(z - lse)
    q = p.clone()
    q[torch.arange(n, device=DEV), at] -= 1.0
    slope = 1 - (z / c) ** 2 if c else torch.ones_like(z)
    gr = torch.where(live, gl, 0.0).unsqueeze(1)
    d = gr * q * slope
    dq = p * r + 4 * U32  # 4 U32: the subtraction of the target's 1, and products
    dd = gr.abs() * (dq * slope.abs() + (q.abs() * 2 * (Z / c + 2.0**-22) if c else 0.0)) + HALF_ULP[dtype] * d.abs()
    dd = dd * 1.01 + 4 * U32 * d.abs()
    dx, dw = d @ w, d.t() @ x
    bx = dd @ w.abs() + 2 * (vocab + 8) * U32 * (d.abs() @ w.abs()) + HALF_ULP[dtype] * dx.abs() * 1.02 + LEAST
    bw = dd.t() @ x.abs() + 2 * n * U32 * (d.abs().t() @ x.abs()) + HALF_ULP[dtype] * dw.abs() * 1.02 + LEAST
    return (losses, dx, dw), (lb, bx, bw)


def run(x, w, y, gl, softcap=None, **kw):
    x, w = x.detach().to(DEV).requires_grad_(), w.detach().to(DEV).requires_grad_()
    loss = linear_cross_entropy(x, w, y.to(DEV), softcap=softcap, reduction="none", **kw)
    dx, dw = torch.autograd.grad(loss, [x, w], gl.to(DEV))
    return loss.detach(), dx, dw


def within(got, want, bound):
    return bool(((got.double() - want).abs() <= bound).all())


SIZES = [(1, 8, 3), (1, 64, 1000), (2, 520, 1), (3, 40, 257), (17, 33, 511), (64, 128, 256), (255, 72, 300),
         (256, 256, 512), (257, 264, 1025), (300, 1000, 2999), (513, 96, 5000), (65, 4096, 999), (1030, 48, 130)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,width,vocab", SIZES)
@pytest.mark.parametrize("softcap", [None, 5.0])
def test_losses_and_gradients(n, width, vocab, softcap, dtype):
    x, w, y, gl = inputs(n, width, vocab, dtype, seed=n + width)
    want, bound = reference(x, w, y, gl, softcap, dtype)
    got = run(x, w, y, gl, softcap)
    for a, b, c in zip(got, want, bound):
        assert within(a, b, c)
    again = run(x, w, y.int(), gl, softcap)
    for a, b in zip(got, again):
        assert torch.equal(a, b)  # int32 targets, and the same bits every time


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_pieces_of_the_vocabulary(dtype, monkeypatch):
    x, w, y, gl = inputs(70, 96, 2050, dtype, seed=4)
    y[:4] = torch.tensor([255, 256, 511, 512])  # at the pieces' edges
    want, bound = reference(x, w, y, gl, None, dtype)
    for size in (1, 70 * 2 * 512, 70 * 4 * 1024):
        monkeypatch.setattr(vocabulary, "PIECE_BYTES", size)
        for a, b, c in zip(run(x, w, y, gl), want, bound):
            assert within(a, b, c)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_large_logits(dtype):
    """Logits of hundreds: no overflow, probabilities of 0 and 1."""
    x, w, y, gl = inputs(40, 64, 700, dtype, seed=6, size=60.0)
    want, bound = reference(x, w, y, gl, None, dtype)
    got = run(x, w, y, gl)
    for a, b, c in zip(got, want, bound):
        assert torch.isfinite(a).all() and within(a, b, c)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masked_rows(dtype):
    """Ignored rows may hold anything and all rows may be ignored; a target outside the vocabulary is NaN."""
    x, w, y, gl = inputs(40, 64, 300, dtype, seed=8)
    y[3], y[20] = -100, -100
    clean = run(x, w, y, gl)
    x[3], x[20] = math.nan, math.inf
    for a, b in zip(run(x, w, y, gl), clean):
        assert torch.equal(a, b)
    off = torch.full_like(y, -100)
    loss, dx, dw = run(x, w, off, gl)
    assert not loss.any() and not dx.any() and not dw.any()
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    mean = linear_cross_entropy(xd, wd, off.to(DEV))
    assert mean.isnan()
    for t in torch.autograd.grad(mean, [xd, wd]):
        assert not t.any()
    y2 = y.clone()
    y2[7], y2[9] = 300, -1
    loss, dx, dw = run(x, w, y2, gl)
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[7, 9]] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(dx.isnan().any(1), bad)
    assert torch.isfinite(dw).all()


def test_reductions_shapes_and_ignore_index():
    x, w, y, gl = inputs(24, 40, 90, torch.float32, seed=2)
    x3, y3 = x.view(2, 12, 40).to(DEV), y.view(2, 12).to(DEV)
    none = linear_cross_entropy(x3, w.to(DEV), y3, reduction="none")
    assert none.shape == (2, 12) and none.dtype == torch.float32
    total = none.double().sum().float()  # the losses are added in 64 bits and rounded once
    assert torch.equal(linear_cross_entropy(x3, w.to(DEV), y3, reduction="sum"), total)
    assert torch.equal(linear_cross_entropy(x3, w.to(DEV), y3), total / (y3 != -100).sum())
    other = torch.where(y3 == -100, 5, y3)
    ignored = linear_cross_entropy(x3, w.to(DEV), other, ignore_index=5, reduction="none")
    assert torch.equal(ignored == 0, other == 5)
    one = linear_cross_entropy(x3[0, 0], w.to(DEV), torch.tensor(3, device=DEV), reduction="none")
    assert one.shape == ()
    empty = linear_cross_entropy(x3[:0], w.to(DEV), y3[:0], reduction="none")
    assert empty.shape == (0, 12)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layouts(dtype):
    """Pitched, transposed and unaligned inputs give what contiguous ones give."""
    x, w, y, gl = inputs(50, 64, 200, dtype, seed=12)
    base = run(x, w, y, gl)
    wide_x = torch.zeros(50, 150, dtype=dtype)
    wide_w = torch.zeros(200, 201, dtype=dtype)
    wide_x[:, 3:67], wide_w[:, 1:65] = x, w
    xs = wide_x.to(DEV)[:, 3:67]
    ws = wide_w.to(DEV)[:, 1:65]
    xt = x.to(DEV).t().contiguous().t()
    wt = w.to(DEV).t().contiguous().t()
    for a, b in ((xs, ws), (xt, wt)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        loss = linear_cross_entropy(a, b, y.to(DEV), reduction="none")
        got = (loss.detach(), *torch.autograd.grad(loss, [a, b], gl.to(DEV)))
        for p, q in zip(got, base):
            assert torch.equal(p, q)


def test_gradient_against_differences():
    x, w, y, gl = inputs(30, 48, 120, torch.float32, seed=15)
    _, dx, dw = run(x, w, y, gl, 8.0)
    g = torch.Generator().manual_seed(1)
    sx, sw = torch.randn(x.shape, generator=g), torch.randn(w.shape, generator=g) / math.sqrt(48)
    h = 2.0**-9

    def f(k):
        loss = linear_cross_entropy((x + k * sx).to(DEV), (w + k * sw).to(DEV), y.to(DEV), softcap=8.0,
                                    reduction="none")
        return float((loss.double().cpu() * gl.double()).sum())

    got = (f(h) - f(-h)) / (2 * h)
    want = float((dx.double().cpu() * sx.double()).sum() + (dw.double().cpu() * sw.double()).sum())
    # A loss of about 5 to 1e-6, over the step, and the third derivative's h^2.
    size = float(gl.double().abs().sum())
    assert abs(got - want) <= size * (2e-6 / h + 50 * h * h)


def test_refusals():
    x, w, y = torch.randn(4, 16, device=DEV), torch.randn(9, 16, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for args, kw, err in (((x, w[:, :8], y), {}, ValueError), ((x, w, y[:3]), {}, ValueError),
                          ((x, w, y.float()), {}, TypeError), ((x.half(), w.half(), y), {}, TypeError),
                          ((x.bfloat16(), w, y), {}, TypeError), ((x, w, y), {"reduction": "max"}, ValueError),
                          ((x, w, y), {"softcap": -1.0}, ValueError), ((x, w, y), {"softcap": math.inf}, ValueError),
                          ((x, w.cpu(), y), {}, RuntimeError), ((x.cpu(), w.cpu(), y.cpu()), {}, RuntimeError)):
        with pytest.raises(err):
            linear_cross_entropy(*args, **kw)


def test_other_stream():
    x, w, y, gl = inputs(90, 64, 400, torch.bfloat16, seed=3)
    base = run(x, w, y, gl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, y, gl)
    side.synchronize()
    for a, b in zip(got, base):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# Per example
# ---------------------------------------------------------------------------


def plain_loss(h, w, t):
    live = t != -100
    z = (h @ w.t()).float()
    lse = torch.logsumexp(z, -1)
    zt = z.gather(-1, torch.where(live, t, 0).unsqueeze(-1)).squeeze(-1)
    return (torch.where(live, lse - zt, 0.0)).sum() / live.sum()


@pytest.mark.parametrize("vocab,width", [(61, 24), (64, 40)])
@pytest.mark.parametrize("train", ["head", "table", "both", "tied"])
def test_language_model_under_clipped_grad(train, vocab, width):
    """A model of embedding, one linear layer and the loss, each part trainable."""
    g = torch.Generator().manual_seed(31)
    n, T = 5, 9
    all_params = {"table": torch.randn(vocab, width, generator=g), "mid": torch.randn(width, width, generator=g) / 4,
                  "head": torch.randn(vocab, width, generator=g) / 3}
    names = {"head": ["mid", "head"], "table": ["table", "mid"], "both": ["table", "mid", "head"],
             "tied": ["table", "mid"]}[train]
    y = torch.randint(0, vocab, (n, T), generator=g)
    t = torch.randint(0, vocab, (n, T), generator=g)
    t[:, :3] = -100

    def make(embed, ce, frozen):
        def loss(p, yi, ti):
            q = {**frozen, **p}
            h = torch.tanh(embed(yi, q["table"]) @ q["mid"].t())
            return ce(h, q["table"] if train == "tied" else q["head"], ti)

        return loss

    params = {k: all_params[k] for k in names}
    frozen = {k: v for k, v in all_params.items() if k not in names}
    ref, raux = dp_ref.clipped_grad(make(lambda a, b: b[a], plain_loss, frozen), params, (y, t), clipping_norm=0.7,
                                    normalize_by=float(n))
    grad_fn, st = clipped_grad(make(embedding, linear_cross_entropy, {k: v.to(DEV) for k, v in frozen.items()}),
                               clipping_norm=0.7, normalize_by=float(n), batch_argnums=(1, 2), return_aux=True)
    on = {k: v.to(DEV) for k, v in params.items()}
    for _ in range(2):  # the second call rebinds the plan
        (got, aux), st = grad_fn(on, y.to(DEV), t.to(DEV), state=st)
        assert float(((aux.grad_norms.double().cpu() - raux["norms"].double())
                      / raux["norms"].double()).abs().max()) < 1e-5
        for k in ref:
            assert float((got.pytree[k].double().cpu() - ref[k].double()).norm() / ref[k].double().norm()) < 1e-5


def test_bfloat16_head_through_the_plan():
    """A bfloat16 head's per-example gradients come from the plan's full-weight kernels, within the framework's
    bfloat16 tolerance of float64."""
    n, T, width, vocab = 4, 24, 64, 328
    x, w, y, _ = inputs(n * T, width, vocab, torch.bfloat16, seed=19)
    x, y = x.view(n, T, width), y.view(n, T)
    y[:, 0] = 5  # every example bears a loss

    def loss(p, xi, yi):
        return linear_cross_entropy(xi, p["head"], yi, reduction="sum")

    grad_fn, st = clipped_grad(loss, clipping_norm=1.0, normalize_by=2.0, batch_argnums=(1, 2), return_aux=True)
    (got, aux), st = grad_fn({"head": w.to(DEV)}, x.to(DEV), y.to(DEV), state=st)
    assert any(i[0] == "lin_norm" for i in grad_fn.engine._plan.launch_info)
    norms, out = [], 0.0
    for i in range(n):
        live = y[i] != -100
        z = x[i].double() @ w.double().t()
        q = torch.softmax(z, 1)
        q[torch.arange(T), torch.where(live, y[i], 0)] -= 1.0
        m = (q * live.unsqueeze(1)).t() @ x[i].double()
        norms.append(float(m.norm()))
        out = out + m * min(1.0, 1.0 / norms[-1])
    norms = torch.tensor(norms, dtype=torch.float64)
    assert float(((aux.grad_norms.double().cpu() - norms) / norms).abs().max()) < 2e-2
    assert float((got.pytree["head"].double().cpu() - out / 2.0).norm() / (out / 2.0).norm()) < 2e-2


def test_token_model_trains():
    """Embedding module and loss under ordinary autograd: a few steps lower the loss."""
    torch.manual_seed(0)
    emb = Embedding(50, 32, scale=math.sqrt(32), device=DEV)
    head = torch.nn.Parameter(torch.randn(50, 32, device=DEV) / 8)
    y = torch.randint(0, 50, (8, 20), device=DEV)
    opt = torch.optim.SGD([*emb.parameters(), head], lr=0.5)
    first = None
    for _ in range(20):
        loss = linear_cross_entropy(emb(y), head, y)
        opt.zero_grad()
        loss.backward()
        opt.step()
        first = float(loss.detach()) if first is None else first
    assert float(loss.detach()) < 0.5 * first


def test_without_the_host_helper(monkeypatch):
    """The Functions with vmap rules take the calls outside torch.func when the helper is missing, with the same bits."""
    x, w, y, gl = inputs(60, 72, 310, torch.bfloat16, seed=23)
    toks = torch.randint(0, 310, (60,), device=DEV)

    def all_of():
        out = list(run(x, w, y, gl, 9.0))
        xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        for reduction in ("sum", "mean"):
            loss = linear_cross_entropy(xd, wd, y.to(DEV), reduction=reduction)
            out += [loss.detach(), *torch.autograd.grad(loss, [xd, wd])]
        e = embedding(toks, wd, scale=3.0, padding_idx=7)
        out += [e.detach(), *torch.autograd.grad(e, [wd], torch.ones_like(e))]
        return out

    base = all_of()
    monkeypatch.setattr(vocabulary, "_host_ready", [None])
    for a, b in zip(all_of(), base):
        assert torch.equal(a, b)


def test_no_second_derivative():
    x, w, y, gl = inputs(8, 16, 30, torch.float32, seed=5, ignored=0.0)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    (dx,) = torch.autograd.grad(linear_cross_entropy(xd, wd, y.to(DEV)).square(), [xd], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), [xd])
    (dw,) = torch.autograd.grad(embedding(y.to(DEV), wd).square().sum(), [wd], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dw.sum(), [wd])


def test_head_changed_before_the_backward():
    x, w, y, gl = inputs(8, 16, 30, torch.float32, seed=5)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV)
    loss = linear_cross_entropy(xd, wd, y.to(DEV))
    wd.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


@pytest.mark.parametrize("n", [1, 5, 300])
@pytest.mark.parametrize("softcap", [None, 20.0])
def test_the_targets_entry_keeps_its_bits_in_dx(n, softcap):
    """dx in bfloat16 takes the target's d in float32: only the other entries' rounding is in its bound."""
    x, w, y, gl = inputs(n, 128, 900, torch.bfloat16, seed=40 + n, ignored=0.0)
    _, dx, _ = run(x, w, y, gl, softcap)
    (_, want, _), _ = reference(x, w, y, gl, softcap, torch.bfloat16)
    # As in reference(), with d's own rounding left out at the targets.
    xd, wd, g = x.double().to(DEV), w.double().to(DEV), gl.double().to(DEV).unsqueeze(1)
    u = xd @ wd.t()
    Z = 2 * 128 * U32 * (xd.abs() @ wd.abs().t()) + (softcap * 2.0**-21 if softcap else 0.0)
    z = softcap * torch.tanh(u / softcap) if softcap else u
    p = torch.softmax(z, 1)
    lse = torch.logsumexp(z, 1, keepdim=True)
    r = Z + Z.max(1, keepdim=True).values + (8 + (z - lse).abs()) * 2.0**-22
    q = p.clone()
    at = (torch.arange(n, device=DEV), y.to(DEV))
    q[at] -= 1.0
    slope = 1 - (z / softcap) ** 2 if softcap else torch.ones_like(z)
    d = g * q * slope
    rounding = 2.0**-8 * d.abs()
    rounding[at] = 2 * U32 * d[at].abs()
    dd = g.abs() * ((p * r + 4 * U32) * slope.abs() + (q.abs() * 2 * (Z / softcap + 2.0**-22) if softcap else 0.0))
    dd = dd * 1.01 + rounding + 4 * U32 * d.abs()
    bound = dd @ wd.abs() + 2 * 908 * U32 * (d.abs() @ wd.abs()) + 2.0**-8 * want.abs() * 1.02 + LEAST
    assert within(dx, want, bound)


def test_small_losses_keep_their_bits():
    """A loss far below its log-sum-exp: off by the logits' error times 1 - p, not by the log-sum-exp's last place."""
    width, vocab = 64, 500
    g = torch.Generator().manual_seed(3)
    w = torch.randn(vocab, width, generator=g) / 8
    y = torch.arange(0, vocab, 50)
    x = w[y] * 60.0  # p(target) near 1
    loss = linear_cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), reduction="none").double()
    xd, wd = x.double().to(DEV), w.double().to(DEV)
    z = xd @ wd.t()
    want = torch.logsumexp(z, 1) - z.gather(1, y.to(DEV).unsqueeze(1)).squeeze(1)
    Z = (2 * width * U32 * (xd.abs() @ wd.abs().t())).max(1).values
    share = 1 - torch.exp(-want)
    bound = share * (2 * Z + 2.0**-18) + 4 * U32  # 4 U32: the sum's rounding at 1, and the logarithm's
    assert float(want.min()) < 0.1 and ((loss - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_in_a_graph(dtype):
    """Loss and gradients replayed from a captured graph, with eager work and new contents between the replays."""
    x, w, y, _ = inputs(90, 64, 700, dtype, seed=77)
    x, w, y = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)

    def step():
        loss = linear_cross_entropy(x, w, y)
        return loss, *torch.autograd.grad(loss, [x, w])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        y.copy_(torch.randint(0, 700, (90,), device=DEV))
        y[: 20 * k] = -100  # another number of tokens bears a loss
        with torch.no_grad():
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,width,vocab", [(1, 64, 1000), (5, 40, 3), (70, 96, 2050), (130, 72, 4097), (300, 40, 9000),
                                           (600, 64, 257), (70, 768, 2050), (130, 800, 4097), (300, 1000, 700),
                                           (600, 776, 257)])
@pytest.mark.parametrize("softcap", [None, 5.0])
def test_kept_logits(n, width, vocab, softcap, dtype, monkeypatch):
    """The forward's logits, kept, give the bits that forming them again gives, in pieces too."""
    x, w, y, gl = inputs(n, width, vocab, dtype, seed=n + 3 * vocab)
    y[0] = vocab - 1
    kept = run(x, w, y, gl, softcap)
    monkeypatch.setattr(vocabulary, "PIECE_BYTES", max(n, 1) * 4 * 512)
    for a, b in zip(kept[:1] + kept[2:], (run(x, w, y, gl, softcap))[:1] + run(x, w, y, gl, softcap)[2:]):
        assert torch.equal(a, b)  # dx: pieces change the order of its sums
    monkeypatch.undo()
    monkeypatch.setattr(vocabulary, "KEEP_BYTES", 0)
    for a, b in zip(kept, run(x, w, y, gl, softcap)):
        assert torch.equal(a, b)


def test_logits_are_kept_up_to_a_size_and_until_the_backward(monkeypatch):
    """KEEP_BYTES bounds what a call holds; without a gradient nothing is held, after the backward neither."""
    n, width, vocab = 512, 1024, 16384
    x, w, y, _ = inputs(n, width, vocab, torch.bfloat16, seed=2)
    x, w, y = x.to(DEV).requires_grad_(), w.to(DEV), y.to(DEV)
    logits = 4 * n * vocab

    def held(**kw):
        before = torch.cuda.memory_allocated()
        loss = linear_cross_entropy(x, w, y, **kw)
        mid = torch.cuda.memory_allocated() - before
        if loss.requires_grad:
            loss.backward()
            x.grad = None
        return mid, torch.cuda.memory_allocated() - before

    held()
    mid, after = held()
    assert mid >= logits and after < logits / 4
    monkeypatch.setattr(vocabulary, "KEEP_BYTES", logits - 1)
    assert held()[0] < logits / 4
    monkeypatch.undo()
    with torch.no_grad():
        assert held()[0] < logits / 4


def test_two_backward_passes_of_one_loss():
    x, w, y, gl = inputs(40, 64, 700, torch.bfloat16, seed=12)
    x, w = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss = linear_cross_entropy(x, w, y.to(DEV))
    first = torch.autograd.grad(loss, [x, w], retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(loss, [x, w])):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, [x, w])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,width,vocab", [(2048, 40, 100), (4100, 264, 300), (20000, 24, 70)])
def test_many_tokens_of_a_small_vocabulary(n, width, vocab, dtype, monkeypatch):
    """dW's contraction over the tokens in slices."""
    assert vocabulary._dw_words(vocabulary.dtype_code(dtype), n, vocab, width) > 0
    x, w, y, gl = inputs(n, width, vocab, dtype, seed=n)
    want, bound = reference(x, w, y, gl, None, dtype)
    got = run(x, w, y, gl)
    for a, b, c in zip(got, want, bound):
        assert within(a, b, c)
    for a, b in zip(got, run(x, w, y, gl)):
        assert torch.equal(a, b)
    monkeypatch.setattr(vocabulary, "PIECE_BYTES", 1)
    for a, b, c in zip(run(x, w, y, gl), want, bound):
        assert within(a, b, c)
    monkeypatch.undo()
    few = torch.full_like(y, -100)
    few[n // 2] = vocab - 1
    want, bound = reference(x, w, few, gl, None, dtype)
    for a, b, c in zip(run(x, w, few, gl), want, bound):
        assert within(a, b, c)
    few[n // 2] = -100
    assert not run(x, w, few, gl)[2].any()


def test_frozen_head_under_clipped_grad_with_and_without_kept_logits(monkeypatch):
    g = torch.Generator().manual_seed(7)
    width, vocab, n, T = 136, 700, 4, 8
    w = (torch.randn(vocab, width, generator=g) / 4).to(DEV)
    mid = {"mid": (torch.randn(width, width, generator=g) / 8).to(DEV)}
    x, t = torch.randn(n, T, width, generator=g).to(DEV), torch.randint(0, vocab, (n, T), generator=g).to(DEV)

    def step():
        f, st = clipped_grad(lambda p, xi, ti: linear_cross_entropy(torch.tanh(xi @ p["mid"].t()), w, ti),
                             clipping_norm=0.1, normalize_by=float(n), batch_argnums=(1, 2), return_aux=True)
        (got, aux), _ = f(mid, x, t, state=st)
        return got.pytree["mid"], aux.grad_norms

    kept = step()
    monkeypatch.setattr(vocabulary, "KEEP_BYTES", 0)
    for a, b in zip(kept, step()):
        assert torch.equal(a, b)
    ref, raux = dp_ref.clipped_grad(lambda p, xi, ti: plain_loss(torch.tanh(xi @ p["mid"].t()), w.cpu(), ti),
                                    {"mid": mid["mid"].cpu()}, (x.cpu(), t.cpu()), clipping_norm=0.1,
                                    normalize_by=float(n))
    assert float((kept[0].double().cpu() - ref["mid"].double()).norm() / ref["mid"].double().norm()) < 1e-5
    assert float(((kept[1].double().cpu() - raux["norms"].double()) / raux["norms"].double()).abs().max()) < 1e-5


@pytest.mark.parametrize("outside", [False, True])
def test_gradients_under_vmap(outside):
    """vmap(grad), of inputs that want a gradient outside it too."""
    x, w, y, _ = inputs(12, 136, 300, torch.float32, seed=3, ignored=0.0)
    x, y = x.reshape(3, 4, 136), y.reshape(3, 4)
    xd, wd, yd = x.to(DEV).requires_grad_(outside), w.to(DEV), y.to(DEV)
    got = torch.func.vmap(torch.func.grad(lambda a, b: linear_cross_entropy(a, wd, b, reduction="sum")))(xd, yd)
    want, bound = reference(x.reshape(12, 136), w, y.reshape(12), torch.ones(12), None, torch.float32)
    assert within(got.detach().reshape(12, 136), want[1], bound[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,width,vocab", [(300, 768, 700), (2100, 136, 300), (20, 136, 2000)])
def test_in_a_graph_with_kept_logits_and_slices(n, width, vocab, dtype):
    x, w, y, _ = inputs(n, width, vocab, dtype, seed=78)
    x, w, y = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)

    def step():
        loss = linear_cross_entropy(x, w, y)
        return loss, *torch.autograd.grad(loss, [x, w])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        y.copy_(torch.randint(0, vocab, (n,), device=DEV))
        y[: 4 * k] = -100
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach())


def test_offsets_past_32_bits():
    """A head of 4.9 GB: its last rows are read, and their gradients written, where they lie."""
    n, width, vocab = 24, 1024, 2400000
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randn(vocab, width, generator=g, device=DEV, dtype=torch.bfloat16) / 32
    x = torch.randn(n, width, generator=g, device=DEV, dtype=torch.bfloat16)
    y = torch.tensor([vocab - 1, 0, vocab // 2, vocab - 257] * 6, device=DEV)
    x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), [x, w])
    with torch.no_grad():
        z = torch.cat([x.double() @ p.double().t() for p in w.split(200000)], 1)
        lse = torch.logsumexp(z, 1)
        want = lse - z.gather(1, y.unsqueeze(1)).squeeze(1)
        # float32 sums of `width` products and of the exponentials.
        slack = 4 * width * U32 * (x.double().abs() @ w[y].double().abs().t()).max() + 64 * U32 * lse.abs().max()
        assert float((loss.double() - want).abs().max()) <= float(slack)
        d = torch.softmax(z, 1)
        d[torch.arange(n, device=DEV), y] -= 1.0
        for row in (0, vocab // 2, vocab - 257, vocab - 1):
            exact = d[:, row] @ x.double()
            scale = d[:, row].abs() @ x.double().abs()
            assert bool(((dw[row].double() - exact).abs() <= 2.0**-7 * scale).all())
        near = sum(d[:, k : k + 200000] @ w[k : k + 200000].double() for k in range(0, vocab, 200000))
        size = sum(d[:, k : k + 200000].abs() @ w[k : k + 200000].double().abs() for k in range(0, vocab, 200000))
        assert bool(((dx.double() - near).abs() <= 2.0**-7 * size).all())
