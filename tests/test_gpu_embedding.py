"""The embedding operator: lookup, table gradient, per-example norms and clipped sum.

Checked against plain float64 sums.  A float32 sum of k terms x_j in any order
is off by at most (k - 1) 2^-24 sum|x_j| (1 + small); every product adds one
more 2^-24, the store in the table's type one half ulp of it.  The bounds
below are those, entry by entry.
"""

from __future__ import annotations

import math

import pytest
import torch

from opaque_amd import _native as N
from opaque_amd.clipping import clipped_grad, per_group
from opaque_amd.engine import ClipSpec, EmbeddingSite, GhostPlan, LeafOut, Segments, plan_key
from opaque_amd.guard import guard_constants, leaf_guards
from opaque_amd.vocabulary import Embedding, embedding
from oracle import dp_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0**-24
# Half an ulp of a stored value, and the least subnormal's half.
HALF_ULP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def tokens_of(kind: str, n: int, vocab: int, g: torch.Generator) -> torch.Tensor:
    if kind == "same":
        return torch.full((n,), vocab - 1)
    if kind == "text":  # the log of the token id is uniform
        return (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(vocab + 1)) - 1).long() \
            .clamp(0, vocab - 1)
    y = torch.randint(0, vocab, (n,), generator=g)
    if kind == "padded":
        y[n // 3 :] = 0
    return y


def table_sums(y: torch.Tensor, g: torch.Tensor, vocab: int):
    """float64 sums and sums of magnitudes per token, and each token's count."""
    g64 = g.double().cpu()
    s = torch.zeros(vocab, g.shape[1], dtype=torch.float64).index_add_(0, y, g64)
    m = torch.zeros(vocab, g.shape[1], dtype=torch.float64).index_add_(0, y, g64.abs())
    k = torch.zeros(vocab, dtype=torch.float64).index_add_(0, y, torch.ones(y.numel(), dtype=torch.float64))
    return s, m, k


SIZES = [(1, 8, 5), (2, 1, 1), (31, 33, 7), (32, 64, 40), (33, 65, 3), (64, 512, 1000), (257, 321, 513),
         (1000, 96, 70000), (8192, 40, 511), (8193, 24, 512), (20000, 16, 300000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,width,vocab", SIZES)
@pytest.mark.parametrize("scale", [1.0, -3.3])
def test_lookup_is_one_rounded_product(n, width, vocab, dtype, scale):
    g = gen(n + width)
    w = torch.randn(vocab, width, generator=g).to(dtype).to(DEV)
    y = tokens_of("random", n, vocab, g).to(DEV)
    out = embedding(y, w, scale=scale)
    want = (w[y].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype) if scale != 1.0 else w[y]
    assert torch.equal(out, want)
    assert torch.equal(embedding(y.int(), w, scale=scale), out)


@pytest.mark.parametrize("kind", ["random", "text", "same", "padded"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,width,vocab", SIZES)
def test_table_gradient(n, width, vocab, dtype, kind):
    g = gen(7 * n + width)
    y = tokens_of(kind, n, vocab, g)
    w = torch.randn(vocab, width, generator=g).to(dtype).to(DEV).requires_grad_()
    go = torch.randn(n, width, generator=g).to(dtype).to(DEV)
    scale = 1.75
    (dw,) = torch.autograd.grad(embedding(y.to(DEV), w, scale=scale), w, go)
    s, m, k = table_sums(y, go, vocab)
    bound = (k.unsqueeze(1) + 1) * U32 * 1.001 * scale * m + HALF_ULP[dtype] * 1.001 * (scale * s).abs() \
        + LEAST[dtype]
    bound[k == 0] = 0.0
    assert ((dw.double().cpu() - scale * s).abs() <= bound).all()
    (again,) = torch.autograd.grad(embedding(y.to(DEV), w, scale=scale), w, go)
    assert torch.equal(dw, again)  # no order of execution in the sums


def test_gradient_against_differences():
    g = gen(3)
    w = torch.randn(11, 24, generator=g).to(DEV).requires_grad_()
    y = torch.randint(0, 11, (3, 13), generator=g).to(DEV)
    c = torch.randn(3, 13, 24, generator=g).to(DEV)
    step = torch.randn(11, 24, generator=g).to(DEV)

    def f(t):
        return (embedding(y, t, scale=0.5).double() * c.double()).sum()

    (dw,) = torch.autograd.grad((embedding(y, w, scale=0.5) * c).sum(), w)
    h = 2.0**-6  # the lookup is linear: a difference has only float32 rounding in it
    with torch.no_grad():
        got = float((f(w + h * step) - f(w - h * step)) / (2 * h))
    want = float((dw.double() * step.double()).sum())
    size = float((c.abs().double() * 0.5 * (w.abs() + step.abs())[y].double()).sum())
    assert abs(got - want) <= 4 * U32 * size / h


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layouts(dtype):
    """Pitched, transposed, unaligned and expanded tensors give what contiguous ones give."""
    g = gen(5)
    n, width, vocab = 70, 48, 90
    y = torch.randint(0, vocab, (n,), generator=g).to(DEV)
    big = torch.randn(vocab, 2 * width + 2, generator=g).to(dtype).to(DEV)
    go = torch.randn(n, 2 * width + 2, generator=g).to(dtype).to(DEV)
    for w, d in ((big[:, 1 : 1 + width], go[:, 1 : 1 + width]), (big[:, :width], go[:, width : 2 * width]),
                 (big.t()[:vocab, :width] if big.shape[1] >= vocab else big[:, :width], go[:1, :width].expand(n, width))):
        yy = y % w.shape[0]
        a = w.detach().requires_grad_()
        b = w.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        oa, ob = embedding(yy, a), embedding(yy, b)
        assert torch.equal(oa, ob)
        (ga,), (gb,) = torch.autograd.grad(oa, a, d), torch.autograd.grad(ob, b, d.contiguous())
        assert torch.equal(ga, gb)


def test_tokens_outside_the_table_and_padding():
    w = torch.randn(10, 16, device=DEV, requires_grad=True)
    y = torch.tensor([[-1, 3, 10], [3, 2**40, 5]], device=DEV)
    out = embedding(y, w, padding_idx=5)
    bad = torch.tensor([[True, False, True], [False, True, False]], device=DEV)
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(out[1, 2], w[5])
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    want = torch.zeros(10, 16, device=DEV)
    want[3] = 2.0
    assert torch.equal(dw, want)


def test_empty_and_refusals():
    w = torch.randn(10, 16, device=DEV, requires_grad=True)
    out = embedding(torch.zeros(0, 4, dtype=torch.int64, device=DEV), w)
    assert out.shape == (0, 4, 16)
    (dw,) = torch.autograd.grad(out, w, torch.zeros_like(out))
    assert torch.equal(dw, torch.zeros_like(w))
    y = torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError):
        embedding(y.float(), w)
    with pytest.raises(TypeError):
        embedding(y, w.double())
    with pytest.raises(ValueError):
        embedding(y, w[0])
    with pytest.raises(ValueError):
        embedding(y, w, padding_idx=10)
    with pytest.raises(ValueError):
        embedding(y, w, scale=math.inf)
    with pytest.raises(RuntimeError):
        embedding(y, w.cpu())
    with pytest.raises(RuntimeError):
        embedding(y.cpu(), w)


def test_module_and_other_stream():
    m = Embedding(50, 32, padding_idx=0, scale=2.0, device=DEV)
    y = torch.randint(0, 50, (4, 6), device=DEV)
    want = m(y)
    assert torch.equal(want, (2.0 * m.weight[y]).detach())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = m(y)
        (dw,) = torch.autograd.grad(out, m.weight, torch.ones_like(out))
    torch.cuda.current_stream().wait_stream(side)
    (here,) = torch.autograd.grad(want, m.weight, torch.ones_like(want))
    assert torch.equal(out, want) and torch.equal(dw, here) and not dw[0].any()


# ---------------------------------------------------------------------------
# Per-example norms and the clipped sum
# ---------------------------------------------------------------------------


def clip_of(shape, dtype, thresholds=(1.0,), normalize_by=4.0):
    _, rnd = leaf_guards([shape], [dtype])
    return ClipSpec(mode=N.CLIP_FIXED, thresholds=list(thresholds), effective=float(thresholds[0]),
                    normalize_by=normalize_by, guards=[(*guard_constants(dtype, rnd), dtype)])


def per_example(y, g, lengths, seq, vocab, padding=-1):
    """float64 S, sums of magnitudes and the largest count per (example, token)."""
    S, M, K = [], [], 0.0
    for i, ln in enumerate(lengths):
        yi, gi = y[i * seq : i * seq + ln], g[i * seq : i * seq + ln]
        keep = (yi >= 0) & (yi < vocab) & (yi != padding)
        s, m, k = table_sums(yi[keep], gi[keep], vocab)
        S.append(s)
        M.append(m)
        K = max(K, float(k.max()))
    return torch.stack(S), torch.stack(M), K


CLIPS = [(1, 1, 8, 3, "random"), (3, 5, 24, 4, "random"), (4, 33, 520, 20, "text"), (5, 64, 33, 7, "padded"),
         (2, 200, 16, 9, "same"), (7, 31, 1030, 600, "padded"), (16, 96, 40, 5000, "text")]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("batch,seq,width,vocab,kind", CLIPS)
@pytest.mark.parametrize("second", [False, True])
def test_clipped_sum(batch, seq, width, vocab, kind, dtype, second):
    g = gen(batch * seq + width)
    y = tokens_of(kind, batch * seq, vocab, g)
    go = (torch.randn(batch * seq, width, generator=g)
          * torch.exp(torch.randn(batch, generator=g)).repeat_interleave(seq).unsqueeze(1)
          / math.sqrt(seq * width)).to(dtype)
    lengths = [(seq * (i % 4 + 1) + 3) // 4 if i else seq for i in range(batch)]
    if batch > 2:
        lengths[2] = 0
    scale, padding, nb = 1.5, 1, 4.0
    shape = (vocab, width)
    clip = clip_of(shape, dtype, normalize_by=nb)
    site = EmbeddingSite(tokens=y.to(DEV), g=go.to(DEV), w_leaf=0, scale=scale, padding=padding)
    plan = GhostPlan(segments=Segments.padded(batch, seq, lengths), leaves=[LeafOut(shape, dtype)], clip=clip,
                     embedding_sites=[site], second_moment=second)
    res = plan.run()
    S, M, K = per_example(y, go, lengths, seq, vocab, padding)
    S, M = scale * S, scale * M
    norms = S.flatten(1).norm(dim=1)
    # A norm is off by at most the norm of its entries' errors, its float32
    # squares' roundings and its own store.
    assert ((res.norms.double().cpu() - norms).abs()
            <= (K + 1) * U32 * 1.001 * M.flatten(1).norm(dim=1) + 2 * U32 * 1.001 * norms + 1e-44).all()
    c = res.scales[0, 0].cpu().float().double().view(-1, 1, 1)
    k_all = float(K * batch + batch + 4)
    for got, terms, size in ((res.leaves[0], c * S, c * M),
                             (res.second_moment[0], (c * S) ** 2, (c * M) ** 2) if second else
                             (res.leaves[0], c * S, c * M)):
        want = terms.sum(0) / nb
        bound = 2 * k_all * U32 * size.sum(0) / nb + HALF_ULP[dtype] * 1.001 * want.abs() + LEAST[dtype]
        bound[size.sum(0) == 0] = 0.0
        assert ((got.double().cpu() - want).abs() <= bound).all()
    # New inputs through the same plan, and the same inputs again.
    first = res.leaves[0].clone()
    site2 = EmbeddingSite(tokens=y.flip(0).to(DEV), g=go.to(DEV), w_leaf=0, scale=scale, padding=padding)
    key = plan_key(segments=plan.segments, leaves=plan.leaves, clip=clip, embedding_sites=[site2], device=DEV,
                   second_moment=second)
    assert key == plan.key and plan.rebind(embedding_sites=[site2], clip=clip, key=key)
    plan.run()
    assert plan.rebind(embedding_sites=[site], clip=clip)
    assert torch.equal(plan.run().leaves[0], first)


def test_nonfinite_entries_are_dropped_per_example():
    """An entry of an example's S that is not finite counts as 0, in its norm and in the sum."""
    vocab, width, seq = 6, 40, 70
    g = gen(9)
    y = torch.randint(0, 2, (2 * seq,), generator=g)
    go = torch.randn(2 * seq, width, generator=g)
    go[5, 3] = math.nan
    go[40, 7] = math.inf
    go[60, 7] = -math.inf
    go[80, 11], go[81, 11] = 3e38, 3e38  # their sum overflows float32
    y[80] = y[81] = 4
    y[[5, 40, 60]] = 0
    clip = clip_of((vocab, width), torch.float32)
    plan = GhostPlan(segments=Segments.padded(2, seq), leaves=[LeafOut((vocab, width), torch.float32)], clip=clip,
                     embedding_sites=[EmbeddingSite(tokens=y.to(DEV), g=go.to(DEV), w_leaf=0)])
    res = plan.run()
    S, M, K = per_example(y, go, [seq, seq], seq, vocab)
    keep = torch.ones_like(S, dtype=torch.bool)
    keep[0, 0, 3] = keep[0, 0, 7] = keep[1, 4, 11] = False
    S = torch.where(keep, S, 0.0)
    M = torch.where(keep, M, 0.0)
    norms = S.flatten(1).norm(dim=1)
    assert ((res.norms.double().cpu() - norms).abs() <= (K + 4) * U32 * M.flatten(1).norm(dim=1)).all()
    c = res.scales[0, 0].cpu().float().double().view(-1, 1, 1)
    want = (c * S).sum(0) / clip.normalize_by
    assert ((res.leaves[0].double().cpu() - want).abs()
            <= (2 * K + 8) * U32 * (c * M).sum(0) / clip.normalize_by + LEAST[torch.float32]).all()
    assert not bool(plan.linear_finite())


def test_site_refusals():
    y, go = torch.zeros(8, dtype=torch.int64, device=DEV), torch.zeros(8, 16, device=DEV)
    kw = dict(segments=Segments.padded(2, 4), leaves=[LeafOut((5, 16), torch.float32)],
              clip=clip_of((5, 16), torch.float32))
    for site, err in ((EmbeddingSite(y[:7], go, 0), ValueError), (EmbeddingSite(y, go[:, :8], 0), ValueError),
                      (EmbeddingSite(y.float(), go, 0), TypeError), (EmbeddingSite(y, go.double(), 0), TypeError),
                      (EmbeddingSite(y.cpu(), go, 0), ValueError)):
        with pytest.raises(err):
            GhostPlan(embedding_sites=[site], **kw)
    site = EmbeddingSite(y, go, 0)
    with pytest.raises(ValueError):
        GhostPlan(embedding_sites=[site, site], **kw)


# ---------------------------------------------------------------------------
# Through clipped_grad
# ---------------------------------------------------------------------------


def make_loss(embed):
    def loss(p, y, c):
        h = embed(y, p["table"]) + p["bias"]
        return (torch.tanh(h) * c).sum()

    return loss


def plain(y, w):
    return 2.0 * w[y]


def seam(y, w):
    return embedding(y, w, scale=2.0)


@pytest.mark.parametrize("groups", [False, True])
@pytest.mark.parametrize("microbatch", [None, 2])
@pytest.mark.parametrize("double", [False, True])
def test_clipped_grad_routes_the_table(groups, microbatch, double):
    g = gen(21)
    n, T, vocab, width = 5, 37, 60, 24
    params = {"table": torch.randn(vocab, width, generator=g), "bias": torch.randn(width, generator=g)}
    y = tokens_of("text", n * T, vocab, g).view(n, T)
    c = torch.randn(n, T, width, generator=g)
    on = {k: v.to(DEV) for k, v in params.items()}
    norm = per_group(on, table=3.0, bias=2.0) if groups else 4.0
    kw = dict(normalize_by=float(n), batch_argnums=(1, 2), microbatch_size=microbatch)
    if double:
        kw["compute_dtype"] = torch.float64
    grad_fn, st = clipped_grad(make_loss(seam), clipping_norm=norm, return_aux=True, **kw)
    (got, aux), st = grad_fn(on, y.to(DEV), c.to(DEV), state=st)
    assert len(grad_fn.engine._plan._embeds) == (0 if double else 1)
    cpu_norm = per_group(params, table=3.0, bias=2.0) if groups else 4.0
    ref, raux = dp_ref.clipped_grad(make_loss(plain), params, (y, c), clipping_norm=cpu_norm, normalize_by=float(n))
    # The losses and their gradients come from torch on two devices: tanh and
    # its derivative differ by ulps, so the float32 tolerance of the framework's
    # other end-to-end tests applies.
    assert float(((aux.grad_norms.double().cpu() - raux["norms"].double()) / raux["norms"].double()).abs().max()) < 1e-5
    for k in ref:
        assert float((got.pytree[k].double().cpu() - ref[k].double()).norm() / ref[k].double().norm()) < 1e-5
    # Shared tables and vmap(grad) take the dense route and agree.
    def twice(p, yi, ci):
        return make_loss(seam)(p, yi, ci) + (seam(yi, p["table"]) * ci).sum()

    def twice_plain(p, yi, ci):
        return make_loss(plain)(p, yi, ci) + (plain(yi, p["table"]) * ci).sum()

    grad_fn, st = clipped_grad(twice, clipping_norm=norm, **kw)
    got, st = grad_fn(on, y.to(DEV), c.to(DEV), state=st)
    ref, _ = dp_ref.clipped_grad(twice_plain, params, (y, c), clipping_norm=cpu_norm, normalize_by=float(n))
    for k in ref:
        assert float((got.pytree[k].double().cpu() - ref[k].double()).norm() / ref[k].double().norm()) < 1e-5


@pytest.mark.parametrize("n", [2048, 2049, 32768, 32769, 70001])
def test_sort_sizes(n):
    """Either side of the sizes at which the sort changes its launches, with a token run of thousands."""
    g = gen(n)
    vocab, width = 3000, 8
    y = tokens_of("text", n, vocab, g)
    y[n // 4 : n // 2] = 77
    w = torch.zeros(vocab, width, device=DEV, requires_grad=True)
    go = torch.randint(-8, 9, (n, width), generator=g).float()  # sums exact in float32
    (dw,) = torch.autograd.grad(embedding(y.to(DEV), w), w, go.to(DEV))
    s, _, _ = table_sums(y, go, vocab)
    assert torch.equal(dw.double().cpu(), s)
    batch = 3
    seq = n // batch
    clip = clip_of((vocab, width), torch.float32)
    plan = GhostPlan(segments=Segments.padded(batch, seq), leaves=[LeafOut((vocab, width), torch.float32)], clip=clip,
                     embedding_sites=[EmbeddingSite(tokens=y[: batch * seq].to(DEV), g=go[: batch * seq].to(DEV),
                                                    w_leaf=0)])
    res = plan.run()
    S, _, _ = per_example(y[: batch * seq], go[: batch * seq], [seq] * batch, seq, vocab)
    norms = S.flatten(1).norm(dim=1)
    assert ((res.norms.double().cpu() - norms).abs() <= 4 * U32 * norms).all()  # squares, root and store
    c = res.scales[0, 0].cpu().float().double().view(-1, 1, 1)
    want = (c * S).sum(0) / clip.normalize_by
    bound = 8 * U32 * (c * S).abs().sum(0) / clip.normalize_by + LEAST[torch.float32]
    assert ((res.leaves[0].double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_dropped_rows_may_hold_anything(dtype):
    """Rows of the padding token, of tokens outside the table and outside the segments are not read into any result."""
    g = gen(61)
    batch, seq, width, vocab = 3, 40, 72, 30
    y = torch.randint(0, vocab, (batch * seq,), generator=g)
    go = torch.randn(batch * seq, width, generator=g).to(dtype)
    lengths = [40, 25, 0]
    y[[3, 44]] = 5
    y[[7, 50]] = torch.tensor([vocab, -4])
    drop = (y == 5) | (y < 0) | (y >= vocab)
    inside = torch.cat([torch.arange(seq) < ln for ln in lengths])
    bad = go.clone()
    bad[drop | ~inside] = math.nan
    clip = clip_of((vocab, width), dtype)

    def result(t):
        plan = GhostPlan(segments=Segments.padded(batch, seq, lengths), leaves=[LeafOut((vocab, width), dtype)],
                         clip=clip, embedding_sites=[EmbeddingSite(tokens=y.to(DEV), g=t.to(DEV), w_leaf=0, padding=5)])
        res = plan.run()
        return res.leaves[0], res.norms

    for a, b in zip(result(bad), result(go)):
        assert torch.equal(a, b)
    w = torch.zeros(vocab, width, dtype=dtype, device=DEV, requires_grad=True)
    bad = go.clone()
    bad[drop] = math.inf
    both = [torch.autograd.grad(embedding(y.to(DEV), w, padding_idx=5), w, t.to(DEV))[0] for t in (bad, go)]
    assert torch.equal(*both)


@pytest.mark.parametrize("microbatch", [None, 3])
def test_bfloat16_table_under_clipped_grad(microbatch):
    """A bfloat16 table, whole and in microbatches (whose sums are kept in float32), within the framework's tolerance."""
    g = gen(71)
    n, T, vocab, width = 7, 29, 50, 40
    params = {"table": torch.randn(vocab, width, generator=g).bfloat16()}
    y = tokens_of("text", n * T, vocab, g).view(n, T)
    c = torch.randn(n, T, width, generator=g).bfloat16()

    def loss(embed):
        return lambda p, yi, ci: (embed(yi, p["table"]).float() * ci.float()).sum()

    grad_fn, st = clipped_grad(loss(seam), clipping_norm=30.0, normalize_by=float(n), batch_argnums=(1, 2),
                               return_aux=True, microbatch_size=microbatch)
    (got, aux), st = grad_fn({"table": params["table"].to(DEV)}, y.to(DEV), c.to(DEV), state=st)
    assert got.pytree["table"].dtype == torch.bfloat16
    ref, raux = dp_ref.clipped_grad(loss(plain), params, (y, c), clipping_norm=30.0, normalize_by=float(n))
    assert float(((aux.grad_norms.double().cpu() - raux["norms"].double()) / raux["norms"].double()).abs().max()) < 2e-2
    a, b = got.pytree["table"].double().cpu(), ref["table"].double()
    assert float((a - b).norm() / b.norm()) < 2e-2


def test_in_a_graph():
    """Lookup and table gradient replayed from a captured graph, with eager work and new contents between the replays."""
    vocab, width, n = 700, 48, 300
    w = torch.randn(vocab, width, device=DEV, requires_grad=True)
    y = torch.randint(0, vocab, (n,), device=DEV)
    go = torch.randn(n, width, device=DEV)

    def step():
        out = embedding(y, w, scale=1.5)
        return out, torch.autograd.grad(out, w, go)[0]

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
        go.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach())


def test_offsets_past_32_bits():
    """A table of 4.9 GB: its last rows are read, and their gradients written, where they lie."""
    vocab, width = 2400000, 1024
    w = torch.zeros(vocab, width, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([vocab - 1, 0, vocab - 2, vocab // 2, vocab - 1], device="cuda")
    w[rows] = torch.randn(5, width, device="cuda").to(w.dtype)
    w.requires_grad_()
    out = embedding(rows, w)
    assert torch.equal(out, w.detach()[rows])
    go = torch.randn(5, width, device="cuda").to(w.dtype)
    (dw,) = torch.autograd.grad(out, [w], go)
    assert torch.equal(dw[vocab - 1], (go[0].float() + go[4].float()).to(w.dtype))
    for k in (1, 2, 3):
        assert torch.equal(dw[rows[k]], go[k])
        dw[rows[k]] = 0
    dw[vocab - 1] = 0
    assert not dw.any()
