"""linear_cross_entropy where float32 forms lose bits: loose softcaps, tokens that are nearly certain.

U32 below is 2^-24.  A logit u is a float32 sum of D products, off by at most
Z = 2 D U32 sum|x w|.  A softcapped logit is off by Z and 16 U32 |z| more
(u / c by two roundings, numerator and denominator of the tanh by three each,
the reciprocal's last place and two products, the exponential's argument and
its last place).  The bounds add those, entry by entry, in float64.
"""

from __future__ import annotations

import math

import pytest
import torch

from opaque_amd import vocabulary
from opaque_amd.vocabulary import linear_cross_entropy

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0**-24
HALF_ULP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
LEAST = 2.0**-120


def run(x, w, y, gl, softcap=None):
    x, w = x.detach().to(DEV).requires_grad_(), w.detach().to(DEV).requires_grad_()
    loss = linear_cross_entropy(x, w, y.to(DEV), softcap=softcap, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], gl.to(DEV))
    return loss.detach(), dx, dw


def capped(x, w, y, gl, c, dtype):
    """float64 (losses, dx, dW) under a softcap c, and their bounds."""
    x, w, gl, y = x.double().to(DEV), w.double().to(DEV), gl.double().to(DEV).unsqueeze(1), y.to(DEV)
    n, vocab, width = x.shape[0], w.shape[0], x.shape[1]
    at = (torch.arange(n, device=DEV), y)
    u = x @ w.t()
    z = c * torch.tanh(u / c)
    Z = 2 * width * U32 * (x.abs() @ w.abs().t()) + 16 * U32 * z.abs()
    lse = torch.logsumexp(z, 1, keepdim=True)
    losses = (lse - z[at].unsqueeze(1)).squeeze(1)
    lb = 2 * Z.max(1).values + (16 + losses.abs()) * 2.0**-22 + 4 * U32 * (lse.squeeze(1).abs() + z[at].abs())
    p = torch.exp(z - lse)
    r = Z + Z.max(1, keepdim=True).values + (8 + (z - lse).abs()) * 2.0**-22
    q = p.clone()
    q[at] -= 1.0
    slope, dslope = 1 - (z / c) ** 2, 2 * (z / c).abs() * Z / c + 4 * U32
    d = gl * q * slope
    dd = gl.abs() * ((p * r + 4 * U32) * (slope.abs() + dslope) + q.abs() * dslope) + (HALF_ULP[dtype] + 4 * U32) * d.abs()
    dd = dd * 1.01
    dx, dw = d @ w, d.t() @ x
    bx = dd @ w.abs() + 2 * (vocab + 8) * U32 * (d.abs() @ w.abs()) + HALF_ULP[dtype] * dx.abs() * 1.02 + LEAST
    bw = dd.t() @ x.abs() + 2 * n * U32 * (d.abs().t() @ x.abs()) + HALF_ULP[dtype] * dw.abs() * 1.02 + LEAST
    return (losses, dx, dw), (lb, bx, bw)


CAPS = [0.5, 3.0, 30.0, 1e3, 1e4, 1e6, 1e30]


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cap", CAPS)
def test_softcaps_keep_the_logits_bits(cap, dtype, kept, monkeypatch):
    """Caps from below the logits to far above: the error follows the logit, not the cap."""
    g = torch.Generator().manual_seed(7)
    n, width, vocab = 70, 136, 700
    w = (torch.randn(vocab, width, generator=g) / math.sqrt(width)).to(dtype)
    y = torch.randint(0, vocab, (n,), generator=g)
    x = (torch.randn(n, width, generator=g) + 6.0 * torch.rand(n, 1, generator=g) * w[y].float()).to(dtype)
    gl = torch.randn(n, generator=g)
    if not kept:
        monkeypatch.setattr(vocabulary, "KEEP_BYTES", 0)
    want, bound = capped(x, w, y, gl, cap, dtype)
    for a, b, c in zip(run(x, w, y, gl, cap), want, bound):
        assert ((a.double() - b).abs() <= c).all()


@pytest.mark.parametrize("cap", [1e-3, 30.0, 1e6])
def test_softcaps_at_the_ends(cap):
    """Logits of 0 and far past the cap either way: 0 and the cap itself, and a gradient of the formula's size."""
    w = torch.tensor([[0.0], [1.0], [-1.0], [1e-6]])
    x = torch.tensor([[0.0], [1.0], [1e6 * max(cap, 1.0)], [-1e6 * max(cap, 1.0)]])
    w8, x8 = torch.zeros(4, 8), torch.zeros(4, 8)
    w8[:, :1], x8[:, :1] = w, x
    y = torch.tensor([0, 3, 0, 0])
    want, bound = capped(x8, w8, y, torch.ones(4), cap, torch.float32)
    for a, b, c in zip(run(x8, w8, y, torch.ones(4), cap), want, bound):
        assert torch.isfinite(a).all() and ((a.double() - b).abs() <= c).all()


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("helper", [True, False])
def test_nearly_certain_tokens_keep_their_gradients_bits(dtype, kept, helper, monkeypatch):
    """Tokens of 1 - p(target) from 1e-6 to 1e-1 whose logits are around 500: the target's d = -(1 - p) is off by the
    logits' error times 1 - p and by the roundings of a sum of exponentials near 1 (30 of them), not by the last place
    of the log-sum-exp (1.5e-5)."""
    width, vocab, n = 136, 500, 40
    g = torch.Generator().manual_seed(3)
    w = torch.randn(vocab, width, generator=g) / math.sqrt(width)
    w[:, 0] = 1.0
    y = torch.arange(0, vocab, 13)[:n]
    n = y.numel()
    x = w[y] * torch.linspace(10.0, 22.0, n).unsqueeze(1)
    x[:, 0] = 500.0
    x, w, gl = x.to(dtype), w.to(dtype), torch.linspace(0.5, 2.0, n)
    if not kept:
        monkeypatch.setattr(vocabulary, "KEEP_BYTES", 0)
    if not helper:
        monkeypatch.setattr(vocabulary, "_host_ready", [None])
    loss, dx, dw = run(x, w, y, gl)
    xd, wd, gd, at = x.double().to(DEV), w.double().to(DEV), gl.double().to(DEV).unsqueeze(1), (torch.arange(n), y)
    z = xd @ wd.t()
    lse = torch.logsumexp(z, 1, keepdim=True)
    Z = (2 * width * U32 * (xd.abs() @ wd.abs().t())).max(1, keepdim=True).values
    p = torch.exp(z - lse)
    rest = p.clone()
    rest[at] = 0.0
    share = rest.sum(1)  # 1 - p(target), to float64's relative precision
    assert 1e-7 < float(share.min()) < 1e-5 and float(share.max()) > 1e-2
    q = p.clone()
    q[at] = -share
    dq = p * (2 * Z + (8 + (z - lse).abs()) * 2.0**-22 + 30 * U32)
    dq[at] = share * (2 * Z.squeeze(1) + 48 * 2.0**-22) + 34 * U32
    assert ((loss.double() + torch.log1p(-share)).abs() <= dq[at] / (1 - share)).all()
    d, dd = gd * q, gd * dq * 1.01
    rounding = HALF_ULP[dtype] * d.abs()
    bw = (dd + rounding).t() @ xd.abs() + 2 * n * U32 * (d.abs().t() @ xd.abs()) + HALF_ULP[dtype] * 1.02 * (d.t() @ xd).abs() + LEAST
    rounding[at] = 2 * U32 * d[at].abs()  # dx takes the target's entry in float32
    bx = (dd + rounding) @ wd.abs() + 2 * (vocab + 8) * U32 * (d.abs() @ wd.abs()) + HALF_ULP[dtype] * 1.02 * (d @ wd).abs() + LEAST
    assert ((dx.double() - d @ wd).abs() <= bx).all()
    assert ((dw.double() - d.t() @ xd).abs() <= bw).all()
