"""rms_norm and rms_norm_quantized against the formulas in 64 bits.

Tolerances count roundings: a float32 sum of w squares along the kernel's path (up to 32 additions a thread, then a tree
of at most 10 levels and 16 waves) is off by at most 64 steps of 2^-24 of its value, its root by half of that; a few
more for the products; then half a step of the result's type, ``finfo.eps / 2``.
"""

from __future__ import annotations

import pytest
import torch

from opaque_amd import vocabulary
from opaque_amd.normalization import RMSNorm, rms_norm, rms_norm_quantized

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0**-24
WIDTHS = [1, 3, 8, 31, 64, 65, 128, 200, 256, 257, 512, 515, 1000, 1024, 1032, 2048, 2050, 4096, 4100, 8192, 8193,
          16384, 16391, 32768]


@pytest.fixture(params=[True, False], ids=["helper", "functions"])
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(vocabulary, "_host_ready", [None])


def make(n, width, dtype, stream=None, gain=None, seed=0, groups=None):
    g = torch.Generator().manual_seed(seed + 17 * width + n)
    r = lambda *s: torch.randn(*s, generator=g)
    size = torch.exp(r(n, 1))
    x = (size * r(n, width)).to(dtype).to(DEV)
    res = None if stream is None else (size * r(n, width)).to(stream).to(DEV)
    w = None if gain is None else (1 + 0.3 * r(*((groups,) if groups else ()), width)).to(gain).to(DEV)
    gy = r(n, width).to(dtype).to(DEV)
    gh = None if stream is None else r(n, width).to(stream).to(DEV)
    return x, res, w, gy, gh


def exact(h, w, eps, offset=0.0):
    """(y, u, 1 / sqrt) of stored rows h in 64 bits."""
    h = h.double()
    inv = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    gain = 1.0 if w is None else w.double() + offset
    return h * inv * gain, h * inv, inv


def half(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, bound):
    """|got - want| within bound, element by element."""
    worst = ((got.double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0, worst


def check(x, res, w, gy, gh, eps=1e-6, unit_offset=False):
    ts = [t.detach().requires_grad_() for t in (x, res, w) if t is not None]
    it = iter(ts)
    xl, rl, wl = next(it), next(it) if res is not None else None, next(it) if w is not None else None
    out = rms_norm(xl, wl, residual=rl, eps=eps, unit_offset=unit_offset)
    y, h = out if res is not None else (out, x)
    if res is not None:
        assert h.dtype == res.dtype and torch.equal(h, (x.float() + res.float()).to(res.dtype))
    assert y.dtype == x.dtype and y.shape == x.shape
    offset = 1.0 if unit_offset else 0.0
    want, u, inv = exact(h.detach(), w, eps, offset)
    near(y, want, want.abs() * (40 * U + half(x.dtype)) + torch.finfo(x.dtype).smallest_normal)
    grads = torch.autograd.grad([y, h] if res is not None else [y], ts, [gy, gh] if res is not None else [gy])
    gain = 1.0 if w is None else w.double() + offset
    a = gy.double() * gain
    mean, spread = (a * u).mean(-1, keepdim=True), (a * u).abs().mean(-1, keepdim=True)
    dh = inv * (a - u * mean)
    slack = 100 * U * inv * (a.abs() + u.abs() * spread)
    if gh is not None:
        dh, slack = dh + gh.double(), slack + 4 * U * gh.double().abs()
    dh = dh.expand(x.shape)
    near(grads[0], dh, slack + dh.abs() * half(x.dtype) + torch.finfo(x.dtype).smallest_normal)
    if res is not None:
        assert grads[1].dtype == res.dtype
        near(grads[1], dh, slack + dh.abs() * half(res.dtype) + torch.finfo(res.dtype).smallest_normal)
    if w is not None:
        p = (gy.double() * u).reshape(-1, x.shape[-1])
        dw, size = p.sum(0), p.abs().sum(0)
        assert grads[-1].dtype == w.dtype and grads[-1].shape == w.shape
        near(grads[-1], dw, (p.shape[0] + 64) * U * size + dw.abs() * half(w.dtype)
             + torch.finfo(w.dtype).smallest_normal)
    return y, grads


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_widths(width, dtype):
    check(*make(5, width, dtype, dtype, dtype))


@pytest.mark.parametrize("n", [1, 2, 31, 33, 255, 1025, 4099])
@pytest.mark.parametrize("width", [40, 192, 1001, 2304])
def test_rows(n, width):
    check(*make(n, width, BF16, BF16, BF16))


@pytest.mark.parametrize("types", [(BF16, None, None), (BF16, F32, BF16), (F16, F32, F32), (F32, F32, None),
                                   (F16, F16, F32), (BF16, None, F32), (F32, None, F32)], ids=str)
@pytest.mark.parametrize("width", [100, 768, 4104])
def test_types(path, types, width):
    x, res, w, gy, gh = make(37, width, types[0], types[1], types[2])
    check(x, res, w, gy, gh, eps=1e-5, unit_offset=w is not None and width == 768)


def test_leading_dimensions_and_strides(path):
    """Slices, transposes and expanded gradients: the same bits as their contiguous copies."""
    x, res, w, gy, gh = make(24, 96, BF16, BF16, BF16)
    wide = torch.zeros(24, 131, dtype=BF16, device=DEV)
    wide[:, 3:99] = x
    turned = res.t().contiguous().t()
    gain = torch.zeros(192, dtype=BF16, device=DEV)
    gain[::2] = w
    want = check(x, res, w, gy, gh)
    got = check(wide[:, 3:99], turned, gain[::2], gy.t().contiguous().t(), gh)
    assert torch.equal(want[0], got[0]) and all(torch.equal(a, b) for a, b in zip(want[1], got[1]))
    y, h = rms_norm(x.view(2, 3, 4, 96), w, residual=res.view(2, 3, 4, 96))
    assert torch.equal(y.view(24, 96), want[0]) and y.shape == h.shape == (2, 3, 4, 96)
    assert torch.equal(rms_norm(x[0], w), rms_norm(x[:1], w)[0])
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    one = torch.autograd.grad(rms_norm(x1, w1).sum(), [x1, w1])  # the gradient is one element, expanded
    two = torch.autograd.grad(rms_norm(x1, w1), [x1, w1], torch.ones_like(x1))
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_only_some_gradients(path):
    """Each gradient alone has the bits that all together have; outputs that are not used bring nothing."""
    x, res, w, gy, gh = make(70, 520, F16, F32, F16)
    _, want = check(x, res, w, gy, gh)
    for i in range(3):
        ts = [t.clone() for t in (x, res, w)]
        ts[i].requires_grad_()
        y, h = rms_norm(ts[0], ts[2], residual=ts[1])
        outs = [(o, g) for o, g in ((y, gy), (h, gh)) if o.requires_grad]
        (got,) = torch.autograd.grad([o for o, _ in outs], [ts[i]], [g for _, g in outs])
        assert torch.equal(got, want[i])
    ts = [t.clone().requires_grad_() for t in (x, res, w)]
    y, h = rms_norm(ts[0], ts[2], residual=ts[1])
    a, b, c = torch.autograd.grad(h, ts, gh, retain_graph=True)
    assert torch.equal(a, gh.to(F16)) and torch.equal(b, gh) and not c.any()
    zero = torch.autograd.grad([y, h], ts, [gy, torch.zeros_like(gh)], retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, ts, gy), zero))


def test_differences():
    """The gradients against central differences of the formula in 64 bits."""
    x, res, w, gy, gh = make(3, 12, F32, F32, F32)
    _, grads = check(x, res, w, gy, gh)

    def value(x, r, w):
        h = x + r
        return (exact(h, w, 1e-6)[0] * gy.double()).sum() + (h * gh.double()).sum()

    at = [t.double() for t in (x, res, w)]
    for k, (t, g) in enumerate(zip(at, grads)):
        for i in range(t.numel()):
            step = torch.zeros(t.numel(), dtype=torch.float64, device=DEV)
            step[i] = 1e-5
            up, down = ([*at[:k], t + s * step.view(t.shape), *at[k + 1:]] for s in (1, -1))
            diff = (value(*up) - value(*down)) / 2e-5
            assert abs(diff - g.flatten()[i].double()) < 1e-4 * (1 + abs(diff))


def test_empty_and_special_rows(path):
    """No rows; rows of zeros, infinities, NaN and the largest values touch nothing but themselves."""
    x, _, w, gy, _ = make(9, 100, F32, None, F32)
    leaf, gain = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    y = rms_norm(leaf, gain)
    dx, dw = torch.autograd.grad(y, [leaf, gain], gy[:0])
    assert y.shape == dx.shape == (0, 100) and torch.equal(dw, torch.zeros_like(w))
    clean = rms_norm(x, w)
    x[1], x[3, 5], x[5, 7], x[7] = 0.0, float("inf"), float("nan"), 1e18
    y = rms_norm(x, w)
    assert not y[1].any() and y[3, 5].isnan() and not y[3, :5].any() and y[5].isnan().all()
    assert torch.allclose(y[7], w, rtol=1e-6)
    for i in (0, 2, 4, 6, 8):
        assert torch.equal(y[i], clean[i])
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(rms_norm(leaf, w), [leaf], gy)
    assert dx[[0, 2, 4, 6, 8]].isfinite().all() and dx[5].isnan().all()
    assert torch.allclose(dx[1], gy[1] * w * 1e3, rtol=1e-5)


@pytest.mark.parametrize("width", [24, 500, 4096])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_a_gain_per_example(path, width, dtype):
    """vmap over examples, each with its own gain (what clipped_grad differentiates), one gain for all, and one for
    each of an inner vmap's rows."""
    x, res, _, gy, gh = make(6 * 7, width, dtype, dtype)
    x, res, gy, gh = (t.view(6, 7, width) for t in (x, res, gy, gh))
    g = torch.Generator().manual_seed(3)
    w = (1 + 0.3 * torch.randn(6, width, generator=g)).to(dtype).to(DEV)
    one = lambda x, r, w: rms_norm(x, w, residual=r)
    ts = [t.clone().requires_grad_() for t in (x, res, w)]
    outs = torch.func.vmap(one)(*ts)
    grads = torch.autograd.grad(outs, ts, [gy, gh])
    for i in range(6):
        ti = [t[i].detach().requires_grad_() for t in ts]
        want = one(*ti)
        assert all(torch.equal(o[i], p) for o, p in zip(outs, want))
        for a, b in zip(grads, torch.autograd.grad(want, ti, [gy[i], gh[i]])):
            assert torch.equal(a[i], b)

    def loss(w, x, r, gy, gh):
        y, h = rms_norm(x, w, residual=r)
        return (y * gy).sum() + (h * gh).sum()

    per = torch.func.vmap(torch.func.grad(loss, argnums=(0, 1, 2)), in_dims=(None, 0, 0, 0, 0))(w[0], x, res, gy, gh)
    own = torch.func.vmap(torch.func.grad(loss, argnums=(0, 1, 2)))(w[0].expand(6, -1), x, res, gy, gh)
    assert per[0].shape == (6, width)
    for i in range(6):
        ti = [t.detach().requires_grad_() for t in (w[0], x[i], res[i])]
        want = torch.autograd.grad(one(ti[1], ti[2], ti[0]), ti, [gy[i], gh[i]])
        for a, b, c in zip(per, own, want):
            assert torch.equal(a[i], c) and torch.equal(b[i], c)
    rows = torch.func.vmap(torch.func.vmap(one, in_dims=(0, 0, None)))(x, res, w)
    assert all(torch.equal(a, b) for a, b in zip(rows, outs))
    each = w.unsqueeze(1).expand(6, 7, width).contiguous()
    rows = torch.func.vmap(torch.func.vmap(one))(x, res, each)
    assert all(torch.equal(a, b) for a, b in zip(rows, outs))
    wide = torch.func.vmap(torch.func.vmap(torch.func.grad(loss), in_dims=(None, 0, 0, 0, 0)))(w, x, res, gy, gh)
    want = torch.func.vmap(torch.func.vmap(torch.func.grad(loss)))(each, x, res, gy, gh)
    assert torch.equal(wide, want) and wide.shape == (6, 7, width)


def test_a_rows_result_does_not_depend_on_its_batch():
    """Batches of any size give a row the same bits; repeated calls too."""
    x, res, w, gy, gh = make(2050, 1536, BF16, BF16, BF16)
    y, grads = check(x, res, w, gy, gh)
    y1, grads1 = check(x[70:71], res[70:71], w, gy[70:71], gh[70:71])
    assert torch.equal(y[70:71], y1) and torch.equal(grads[0][70:71], grads1[0])
    for _ in range(3):
        _, again = check(x, res, w, gy, gh)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))


def test_autograd_manners(path):
    x, res, w, gy, gh = make(9, 48, F32, F32, F32)
    ts = [t.requires_grad_() for t in (x, res, w)]
    y, h = rms_norm(x, w, residual=res)
    first = torch.autograd.grad([y, h], ts, [gy, gh], create_graph=True)
    plain = torch.autograd.grad(rms_norm(x, w, residual=res), ts, [gy, gh])
    for d, p in zip(first, plain):
        assert torch.equal(d.detach(), p)
        for t in ts:
            with pytest.raises(RuntimeError):  # NotImplementedError, of the functions
                torch.autograd.grad(d.square().sum(), t, retain_graph=True)
    y, h = rms_norm(x, w, residual=res)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, ts, gy)
    for back in (lambda t: t.cpu(), lambda t: t.double()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            y, h = rms_norm(x, w, residual=res)
        with pytest.raises((RuntimeError, TypeError)):
            torch.autograd.grad([y, h], ts, [gy, gh])
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: turned(t.to(DEV))):
        y, h = rms_norm(x, w, residual=res)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad([y, h], ts, [gy, gh]), plain))
    out = torch.utils.checkpoint.checkpoint(lambda a, b, c: rms_norm(a, c, residual=b), *ts, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, ts, [gy, gh]), plain))
    x.grad = res.grad = None
    y, h = rms_norm(x, w, residual=res)
    torch.autograd.backward([y, h], [gy, gh])
    x.grad.add_(1.0)  # what autograd leaves belongs to each leaf alone
    assert torch.equal(res.grad, plain[1])
    with torch.autograd.forward_ad.dual_level():
        for i in range(3):
            duals = [torch.autograd.forward_ad.make_dual(t.detach(), torch.ones_like(t)) if i == k else t.detach()
                     for k, t in enumerate(ts)]
            with pytest.raises(RuntimeError):
                rms_norm(duals[0], duals[2], residual=duals[1])
    with torch.inference_mode():
        y, h = rms_norm(x.clone(), w.clone(), residual=res.clone())
    assert torch.equal(y, rms_norm(x, w, residual=res)[0])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("width", [1, 64, 100, 128, 136, 500, 1024, 2049, 4096, 8200, 32768])
def test_quantized(dtype, block, width):
    """Scales within their float32 roundings, q the nearest e4m3 values but where the quotient lies on the border
    between two."""
    x, res, w, _, _ = make(6, width, dtype, dtype, dtype)
    x[2], res[2] = 0.0, 0.0
    q, scales, h = rms_norm_quantized(x, w, residual=res, block=block)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    y = exact(h, w, 1e-6)[0]
    size = width if block is None else block
    parts = torch.nn.functional.pad(y, (0, -width % size)).view(6, -1, size)
    want = (parts.abs().amax(2) / 448).clamp_min(torch.finfo(F32).tiny)
    got = scales.view(6, -1).double()
    assert scales.shape == ((6,) if block is None else (6, -(-width // 128)))
    near(got, want, 44 * U * want)
    v = (parts / got.unsqueeze(2)).view(6, -1)[:, :width]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    near(q.to(F32), v, step * 0.5 + 48 * U * v.abs())
    assert q.to(F32).abs().max() <= 448 and not q[2].to(F32).any() and (scales[2] == torch.finfo(F32).tiny).all()


@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("width", [40, 128, 510, 2048])
def test_quantized_borders(path, block, width):
    """Every code of bfloat16 rows: 448 t / max |t| with t = h w is a quotient of 19 bits by 16, a border between two
    codes or 2^-21 away from it, and float32's correct quotient tells which; borders go to the even code."""
    x, res, w, _, _ = make(200, width, BF16, BF16, BF16)
    q, _, h = rms_norm_quantized(x, w, residual=res, block=block)
    t = h.double() * w.double()
    size = width if block is None else block
    parts = torch.nn.functional.pad(t, (0, -width % size)).view(200, -1, size)
    v = (448 * parts / parts.abs().amax(2, keepdim=True)).view(200, -1)[:, :width]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    want = torch.round(v / step) * step
    assert (v / step - torch.floor(v / step) == 0.5).any() or width < 510
    assert torch.equal(q.double(), want)


def test_quantized_values_that_are_none(path):
    x, res, w, _, _ = make(5, 300, F32, F32, F32)
    clean = rms_norm_quantized(x, w, residual=res)
    x[1, 7], x[3, 9] = float("nan"), float("inf")
    q, s, _ = rms_norm_quantized(x, w, residual=res)
    assert s[1].isnan() and q[1].to(F32).isnan().all() and s[3].isnan()
    for i in (0, 2, 4):
        assert torch.equal(q[i].view(torch.uint8), clean[0][i].view(torch.uint8)) and s[i] == clean[1][i]
    big = torch.zeros(2, 300, device=DEV)
    big[:, :3] = torch.tensor([4.0, -1.0, 1e-4], device=DEV)  # of a root mean square of 0.24
    for block in (None, 128):
        q, s = rms_norm_quantized(big, torch.full((300,), 1e38, device=DEV), block=block)
        first = s if block is None else s[:, 0]
        q = q.to(F32)
        assert first.isinf().all() and q[:, 0].isnan().all() and (q[:, 2:128] == 0).all()
        q, s = rms_norm_quantized(big, torch.full((300,), 2e37, device=DEV), block=block)  # the largest y: 3.36e38
        assert s.isfinite().all() and (q.to(F32)[:, 0] == 448).all() and (q.to(F32)[:, 1] == -112).all()
    q, s = rms_norm_quantized(x[:0], w, block=128)
    assert q.shape == (0, 300) and s.shape == (0, 3)


def test_quantized_is_the_norm(path):
    """The same norm as rms_norm's, whichever scales."""
    x, res, w, _, _ = make(40, 640, BF16, F32, BF16)
    y, h = rms_norm(x.float(), w.float(), residual=res)
    for block in (None, 128):
        q, s, h2 = rms_norm_quantized(x, w, residual=res, block=block)
        assert torch.equal(h, h2)
        s = s.unsqueeze(1).expand(40, 640) if block is None else s.repeat_interleave(128, 1)
        assert ((q.to(F32) * s - y).abs() <= y.abs() * 2.0**-4 * (1 + 1e-5) + s * 2.0**-10 * (1 + 1e-5)).all()


def test_under_the_other_transforms(path):
    """grad alone, and what there is no derivative for: jvp, grad of grad."""
    x, res, w, gy, gh = make(4, 40, F32, F32, F32)

    def loss(x, r, w):
        y, h = rms_norm(x, w, residual=r)
        return (y * gy).sum() + (h * gh).sum()

    got = torch.func.grad(loss, argnums=(0, 1, 2))(x, res, w)
    ts = [t.clone().requires_grad_() for t in (x, res, w)]
    y, h = rms_norm(ts[0], ts[2], residual=ts[1])
    for a, b in zip(got, torch.autograd.grad([y, h], ts, [gy, gh])):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda w: torch.func.grad(loss, argnums=2)(x, res, w).square().sum())(w)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: rms_norm(a, w), (x,), (torch.ones_like(x),))
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda a: rms_norm_quantized(a, w)[0])(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_quantized(x, ts[2])
    with torch.no_grad():
        assert rms_norm_quantized(x, ts[2])[0].shape == x.shape


def test_the_same_tensor_twice(path):
    """x as its own residual: its gradient is both parts."""
    x, _, w, gy, _ = make(5, 72, F32, None, F32)
    leaf = x.clone().requires_grad_()
    y, h = rms_norm(leaf, w, residual=leaf)
    (both,) = torch.autograd.grad([y, h], [leaf], [gy, gy])
    ts = [x.clone().requires_grad_(), x.clone().requires_grad_()]
    y, h = rms_norm(ts[0], w, residual=ts[1])
    a, b = torch.autograd.grad([y, h], ts, [gy, gy])
    assert torch.equal(both, a + b)


def test_module():
    m = RMSNorm(200, eps=1e-5, device=DEV, dtype=BF16)
    x, res, _, _, _ = make(4, 200, BF16, BF16)
    assert torch.equal(m(x), rms_norm(x, m.weight, eps=1e-5))
    y, h = m(x, res)
    assert torch.equal(y, rms_norm(x, m.weight, residual=res, eps=1e-5)[0]) and m.weight.requires_grad
    plus = RMSNorm(200, unit_offset=True, device=DEV, dtype=BF16)
    assert not plus.weight.any() and torch.equal(plus(x), rms_norm(x, torch.ones(200, dtype=BF16, device=DEV)))


def test_offsets_past_32_bits():
    """More than 2^32 bytes and 2^31 elements: the last rows have the bits that they have alone."""
    n, width = (1 << 19) + 3, 4104
    x = torch.zeros(n, width, dtype=BF16, device=DEV)
    last, res, w, gy, _ = make(5, width, BF16, BF16, BF16)
    x[-5:] = last
    leaf, gain = last.clone().requires_grad_(), w.clone().requires_grad_()
    want = rms_norm(leaf, gain)
    grads = torch.autograd.grad(want, [leaf, gain], gy)
    x.requires_grad_()
    y = rms_norm(x, gain)
    assert torch.equal(y[-5:], want) and not y[-9:-5].any()
    g = torch.zeros_like(y)
    g[-5:] = gy
    dx, dw = torch.autograd.grad(y, [x, gain], g)
    assert torch.equal(dx[-5:], grads[0]) and not dx[-9:-5].any()
    assert ((dw.double() - grads[1].double()).abs() <= grads[1].double().abs() * 2.0**-7 + 1e-6).all()


def test_on_another_stream():
    x, res, w, gy, gh = make(600, 1024, BF16, BF16, BF16)
    want = check(x, res, w, gy, gh)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = check(x, res, w, gy, gh)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want[1], got[1]))


def test_in_a_graph():
    """Captured once with its gradients, replayed on new values with eager calls between."""
    x, res, w, gy, gh = make(300, 768, BF16, BF16, BF16)
    ts = [t.clone().requires_grad_() for t in (x, res, w)]

    def step():
        y, h = rms_norm(ts[0], ts[2], residual=ts[1])
        q = rms_norm_quantized(ts[0].detach(), ts[2].detach(), block=128)
        return [y.detach(), h.detach(), *q, *torch.autograd.grad([y, h], ts, [gy, gh])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            for t, v in zip(ts, (x, res, w)):
                t.copy_(v * (1 + 0.25 * k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
