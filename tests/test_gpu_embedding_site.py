"""EmbeddingSite through a plan: rebinding, and segments of its own."""

from __future__ import annotations

import pytest
import torch

from opaque_amd import _native as N
from opaque_amd.engine import ClipSpec, EmbeddingSite, GhostPlan, LeafOut, Segments, plan_key
from opaque_amd.guard import guard_constants, leaf_guards

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0**-24


def clip_of(shapes, dtype=torch.float32):
    _, rnd = leaf_guards(shapes, [dtype] * len(shapes))
    return ClipSpec(mode=N.CLIP_FIXED, thresholds=[1.0], effective=1.0, normalize_by=2.0,
                    guards=[(*guard_constants(dtype, rnd), dtype)])


def test_rebind_refuses_tokens_of_another_device():
    """Tokens in host memory are refused as at construction; nothing is launched on them."""
    shape = (9, 16)
    clip = clip_of([shape])
    y, g = torch.randint(0, 9, (12,), device=DEV), torch.randn(12, 16, device=DEV)
    plan = GhostPlan(segments=Segments.padded(3, 4), leaves=[LeafOut(shape, torch.float32)], clip=clip,
                     embedding_sites=[EmbeddingSite(y, g, 0)])
    away = [EmbeddingSite(y.cpu(), g, 0)]
    key = plan_key(segments=plan.segments, leaves=plan.leaves, clip=clip, embedding_sites=away, device=DEV)
    assert key != plan.key
    assert not plan.rebind(embedding_sites=away, clip=clip)
    assert not plan.rebind(embedding_sites=away, clip=clip, key=key)


def test_tables_with_segments_of_their_own():
    """Two tables read at different row counts an example, in one plan (sums of whole numbers: exact in float32)."""
    gen = torch.Generator().manual_seed(3)
    n, rows, shapes = 3, (7, 40), ((11, 24), (300, 8))
    segs = [Segments.padded(n, r, [r, r - 3, 0]) for r in rows]
    ys = [torch.randint(0, s[0], (n * r,), generator=gen) for r, s in zip(rows, shapes)]
    gs = [torch.randint(-8, 9, (n * r, s[1]), generator=gen).float() for r, s in zip(rows, shapes)]
    clip = clip_of(shapes)
    sites = [EmbeddingSite(y.to(DEV), g.to(DEV), k, segments=segs[k] if k else None)
             for k, (y, g) in enumerate(zip(ys, gs))]
    plan = GhostPlan(segments=segs[0], leaves=[LeafOut(s, torch.float32) for s in shapes], clip=clip,
                     embedding_sites=sites)
    res = plan.run()
    S = []
    for y, g, r, s, seg in zip(ys, gs, rows, shapes, segs):
        S.append(torch.stack([torch.zeros(s, dtype=torch.float64).index_add_(0, y[i * r : i * r + ln],
                                                                             g[i * r : i * r + ln].double())
                              for i, ln in enumerate(seg.lengths)]))
    norms = sum(t.flatten(1).square().sum(1) for t in S).sqrt()
    assert ((res.norms.double().cpu() - norms).abs() <= 4 * U32 * norms).all()  # squares, root and store
    c = res.scales[0, 0].cpu().float().double().view(-1, 1, 1)
    for got, t in zip(res.leaves, S):
        bound = 8 * U32 * (c * t).abs().sum(0) / 2.0 + 2.0**-150  # a product, two sums, the quotient and the store
        assert ((got.double().cpu() - (c * t).sum(0) / 2.0).abs() <= bound).all()
