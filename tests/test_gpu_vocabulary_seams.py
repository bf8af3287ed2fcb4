"""Models around the vocabulary operators under clipped_grad: which leaves stay seams, and their values.

Float32 models are held to the framework's end-to-end float32 tolerance (1e-5
of the values' norm, against vmap(grad) on the CPU), bfloat16 ones to its
bfloat16 tolerance (2e-2, against float64).
"""

from __future__ import annotations

import pytest
import torch

from opaque_amd import capture
from opaque_amd.clipping import clipped_grad
from opaque_amd.vocabulary import embedding, linear_cross_entropy
from oracle import dp_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def plain_embedding(y, w, scale=1.0):
    return w[y] if scale == 1.0 else scale * w[y]


def plain_loss(h, w, t):
    z = (h @ w.t()).to(torch.promote_types(h.dtype, torch.float32))
    return (torch.logsumexp(z, -1) - z.gather(-1, t.unsqueeze(-1)).squeeze(-1)).mean()


def compare(make, params, batch, *, tol, steps=2, clipping_norm=0.7, **kw):
    """Clipped sums and norms of ``make(ops)`` against the oracle's in 64 bits; returns the engine."""
    ref, raux = dp_ref.clipped_grad(make(PLAIN), {k: v.double() for k, v in params.items()}, batch,
                                    clipping_norm=clipping_norm, normalize_by=float(len(batch[0])))
    grad_fn, st = clipped_grad(make(OPS), clipping_norm=clipping_norm, normalize_by=float(len(batch[0])),
                               batch_argnums=tuple(range(1, 1 + len(batch))), return_aux=True, **kw)
    on, dev_batch = {k: v.to(DEV) for k, v in params.items()}, [b.to(DEV) for b in batch]
    for _ in range(steps):  # the later calls rebind the plan
        (got, aux), st = grad_fn(on, *dev_batch, state=st)
        assert float(((aux.grad_norms.double().cpu() - raux["norms"].double())
                      / raux["norms"].double()).abs().max()) < tol
        for k in ref:
            a, b = got.pytree[k].double().cpu(), ref[k].double()
            assert float((a - b).norm() / b.norm()) < tol, k
    return grad_fn.engine


class OPS:
    linear = staticmethod(capture.linear)
    embedding = staticmethod(embedding)
    loss = staticmethod(lambda h, w, t: linear_cross_entropy(h, w, t))


class PLAIN:
    linear = staticmethod(torch.nn.functional.linear)
    embedding = staticmethod(plain_embedding)
    loss = staticmethod(plain_loss)


DERIVED = {
    "scaled": lambda w: 0.5 * w,
    "slice": lambda w: w[:40],
    "cast": lambda w: w.double().to(w.dtype),
}


@pytest.mark.parametrize("made", DERIVED)
@pytest.mark.parametrize("which", ["head", "table"])
def test_a_table_tied_to_a_head_made_from_it(made, which):
    """A head that is a cast, a slice or a scaled copy of the embedding table (or a table made from the head): the
    leaf's whole gradient is in its norm and sum."""
    g = torch.Generator().manual_seed(11)
    n, T, vocab, width = 4, 6, 50, 16
    params = {"table": torch.randn(vocab, width, generator=g),
              "mid": torch.randn(width, width, generator=g) / 4}
    y, t = torch.randint(0, 40, (n, T), generator=g), torch.randint(0, 40, (n, T), generator=g)

    def make(ops):
        def loss(p, yi, ti):
            w = p["table"]
            table, head = (w, DERIVED[made](w)) if which == "head" else (DERIVED[made](w), w)
            return ops.loss(torch.tanh(ops.embedding(yi, table)) @ p["mid"].t(), head, ti)

        return loss

    compare(make, params, (y, t), tol=1e-5)


def seams_of(engine):
    """(embedding sites, full-weight sites, whether a leaf is materialised) of the engine's last plan."""
    plan = engine._plan
    return (len(plan._embeds), sum(1 for k in plan._ext_keys if k[0] == "linx"),
            "sqnorm" in {i[0] for i in plan.launch_info})


@pytest.mark.parametrize("microbatch", [None, 2])
def test_seams_of_different_row_counts(microbatch):
    """More hidden rows than tokens (a prefix before them), the loss over the tokens' rows: each seam brings its rows."""
    g = torch.Generator().manual_seed(21)
    n, T, pre, vocab, width = 5, 13, 4, 72, 32
    params = {"table": torch.randn(vocab, width, generator=g), "mid": torch.randn(width, width, generator=g) / 5,
              "head": torch.randn(vocab, width, generator=g) / 5}
    params = {k: v.bfloat16() for k, v in params.items()}
    prefix = torch.randn(pre, width, generator=g).bfloat16()
    y, t = torch.randint(0, vocab, (n, T), generator=g), torch.randint(0, vocab, (n, T), generator=g)

    def make(ops):
        def loss(p, yi, ti):
            h = ops.embedding(yi, p["table"])
            h = torch.cat([prefix.to(h.device, h.dtype), h])
            h = h + torch.tanh(ops.linear(h, p["mid"]))
            h = torch.cat([h[pre:], h[:pre].sum(0, keepdim=True)])[:T]
            return ops.loss(h, p["head"], ti)

        return loss

    engine = compare(make, params, (y, t), tol=2e-2, microbatch_size=microbatch)
    assert seams_of(engine) == (1, 2, False)


def test_a_pooled_head_beside_a_lookup():
    """One lookup of T rows and one linear of one row an example: both are seams, whichever comes first."""
    g = torch.Generator().manual_seed(22)
    n, T, vocab, width, classes = 6, 11, 60, 24, 16
    params = {"table": torch.randn(vocab, width, generator=g).bfloat16(),
              "head": (torch.randn(classes, width, generator=g) / 5).bfloat16()}
    y, c = torch.randint(0, vocab, (n, T), generator=g), torch.randint(0, classes, (n,), generator=g)

    def make(ops):
        def loss(p, yi, ci):
            z = ops.linear(torch.tanh(ops.embedding(yi, p["table"])).mean(0), p["head"])
            z = z.to(torch.promote_types(z.dtype, torch.float32))
            return torch.logsumexp(z, -1) - z.gather(-1, ci.unsqueeze(-1)).squeeze(-1)

        return loss

    assert seams_of(compare(make, params, (y, c), tol=2e-2)) == (1, 1, False)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32], ids=str)
def test_learned_positions_stay_seams(kind):
    """A table read at positions that are the same for every example (not batched under vmap) is a seam, as are the
    model's others, on every step."""
    g = torch.Generator().manual_seed(23)
    n, T, vocab, width = 4, 10, 48, 24
    params = {"wte": torch.randn(vocab, width, generator=g), "wpe": torch.randn(16, width, generator=g),
              "mid": torch.randn(width, width, generator=g) / 4, "head": torch.randn(vocab, width, generator=g) / 4}
    params = {k: v.bfloat16() for k, v in params.items()}
    y, t = torch.randint(0, vocab, (n, T), generator=g), torch.randint(0, vocab, (n, T), generator=g)

    def make(ops):
        def loss(p, yi, ti):
            at = torch.arange(T, device=p["wpe"].device).to(kind)
            h = ops.embedding(yi, p["wte"]) + ops.embedding(at, p["wpe"])
            return ops.loss(torch.tanh(ops.linear(h, p["mid"])), p["head"], ti)

        return loss

    engine = compare(make, params, (y, t), tol=2e-2, steps=3)
    assert seams_of(engine) == (2, 2, False)
    assert engine._discovery is not None and engine.last_rebound


def test_positions_alone():
    """The only table is read at positions: a vector per example, of one row."""
    g = torch.Generator().manual_seed(24)
    params = {"wpe": torch.randn(5, 8, generator=g)}
    x = torch.randn(3, 8, generator=g)

    def make(ops):
        return lambda p, xi: (ops.embedding(torch.tensor(2, device=xi.device), p["wpe"]) * xi).sum().sin()

    assert seams_of(compare(make, params, (x,), tol=1e-5, clipping_norm=10.0)) == (1, 0, False)


@pytest.mark.parametrize("tokens", ["batch", "positions"])
def test_inner_vmaps_of_the_loss(tokens):
    """A loss that vmaps over its own tokens: lookups and losses of the batch are recorded by the engine's vmap, a lookup
    that only the inner one batches is not (the model then goes materialised)."""
    g = torch.Generator().manual_seed(25)
    n, T, vocab, width = 4, 6, 40, 16
    params = {"table": torch.randn(vocab, width, generator=g), "head": torch.randn(vocab, width, generator=g) / 4}
    y, t = torch.randint(0, vocab, (n, T), generator=g), torch.randint(0, vocab, (n, T), generator=g)

    def make(ops):
        def loss(p, yi, ti):
            at = yi if tokens == "batch" else torch.arange(T, device=yi.device)
            h = torch.func.vmap(lambda k: torch.tanh(ops.embedding(k, p["table"])))(at.unsqueeze(1)).squeeze(1)
            h = h * (1 + yi.unsqueeze(1) % 3)
            return torch.func.vmap(lambda r, k: ops.loss(r, p["head"], k))(h, ti).mean()

        return loss

    engine = compare(make, params, (y, t), tol=1e-5)
    assert seams_of(engine)[0] == (1 if tokens == "batch" else 0)
