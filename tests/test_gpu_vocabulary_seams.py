"""Models around the vocabulary operators under clipped_grad: which leaves stay seams, and their values.

Float32 models are held to the framework's end-to-end float32 tolerance (1e-5
of the values' norm, against vmap(grad) on the CPU), bfloat16 ones to its
bfloat16 tolerance (2e-2, against float64).
"""

from __future__ import annotations

import pytest
import torch

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
    embedding = staticmethod(embedding)
    loss = staticmethod(lambda h, w, t: linear_cross_entropy(h, w, t))


class PLAIN:
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
