"""The root-mean-square norm of a block, behind the residual stream's addition.

``rms_norm`` adds a block's output to the stream, norms the sum and hands both
on; its gradients come from one pass over the rows.  Inside ``clipped_grad`` a
gain that trains has a gradient per example ([examples, width], as every leaf
outside the seams): one launch makes them for the whole batch, where
``vmap(grad)`` runs a dozen elementary operations over it
(opaque-engine/.../clipping/_clipped_fun.py:756-762).  ``rms_norm_quantized``
is the same norm in 8 bits with scales, for products that read it so.

The work runs in the HIP kernels of ``libopaque_dp.so`` on the current stream;
there is no CPU route.
"""

from __future__ import annotations

import torch

from opaque_amd import _native as N
from opaque_amd._vmap import front, merged
from opaque_amd.capture import transformed
from opaque_amd.engine import dtype_code
from opaque_amd.vocabulary import _F32, _bound, _call, _OnDevice, _stream, no_tangent, pitched_rows

_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_WIDE = 32768  # the widest row (ODP_NORM_WIDE)
_GRAD_GAINS = 1 << 21  # gains of a call (ODP_NORM_GRAD_GAINS)
BLOCK = 128  # columns of a scale of ``rms_norm_quantized(block=128)``


class _Gain:
    """Gains as the kernels take them: [width], one for all rows, or [groups, width], one for each group of rows."""

    def __init__(self, weight: torch.Tensor | None, groups: int | None, like: torch.Tensor) -> None:
        self.count, self.pitch, self.held, self.dt = 1 if groups is None else groups, 0, None, dtype_code(like.dtype)
        if weight is None:
            return
        w = weight.detach().resolve_neg()
        if w.dim() == 1:
            w = w.contiguous()
        else:
            self.count = w.shape[0]
            if w.stride(0) != 0 or (w.stride(1) != 1 and w.shape[1] > 1):
                w = pitched_rows(w)
                self.pitch = w.stride(0)
        self.held, self.dt = w, dtype_code(w.dtype)


def _forward(x, residual, weight, eps, offset, keep, quant=0):
    """(y, the sum or None, 1 / sqrt(..) or None, scales or None)."""
    rows = pitched_rows(x.detach())
    r = None if residual is None else pitched_rows(residual.detach())
    n, width = rows.shape
    g, dev = _Gain(weight, None, x), x.device
    y = torch.empty(x.shape, dtype=torch.float8_e4m3fn if quant else x.dtype, device=dev)
    h = None if r is None else torch.empty(x.shape, dtype=r.dtype, device=dev)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if keep else None
    lead = x.shape[:-1] if quant != 2 else (*x.shape[:-1], -(-width // BLOCK))
    scales = torch.empty(lead, dtype=torch.float32, device=dev) if quant else None
    at = lambda t: None if t is None else t.data_ptr()
    with _OnDevice(x):
        _call("odp_rms_norm", _stream(x), dtype_code(x.dtype), dtype_code(x.dtype if r is None else r.dtype), g.dt,
              rows.data_ptr(), rows.stride(0), at(r), 0 if r is None else r.stride(0), n, width, at(g.held), g.pitch, g.count,
              eps, offset, quant, y.data_ptr(), at(h), at(rstd), at(scales))
    return y, h, rstd, scales


def _gradients(gy, gh, h, rstd, weight, dtype, offset, groups, need_x, need_r, need_w):
    """(dx, dres, dgain); dgain [width], or one for each of ``groups`` groups of rows (none in an empty batch)."""
    like = gy if gy is not None else gh
    for t in (h, rstd, *(() if weight is None else (weight,))):
        if t.device != like.device:
            raise RuntimeError(f"norm operators: a saved tensor came back on {t.device}, not {like.device}")
    rows = pitched_rows(h.detach())
    n, width = rows.shape
    gy = torch.zeros(h.shape, dtype=dtype, device=h.device) if gy is None else gy
    if gy.dtype != dtype or gy.shape != h.shape or rstd.dtype != torch.float32 or rstd.numel() != n:
        raise RuntimeError("norm operators: a saved tensor came back otherwise than it was saved")
    g = _Gain(weight, groups, gy)
    y2, h2 = pitched_rows(gy.detach()), None if gh is None else pitched_rows(gh.detach())
    same, dev = h.dtype == dtype, h.device
    dx = torch.empty(h.shape, dtype=dtype, device=dev) if need_x or need_r else None
    dr = torch.empty(h.shape, dtype=h.dtype, device=dev) if need_r and not same else None
    dw = words = None
    if need_w:
        make = torch.empty if n else torch.zeros
        dw = make((width,) if groups is None else (groups, width), dtype=weight.dtype, device=dev)
        words = int(N.load().odp_rms_norm_grad_scratch(n, width, g.count))
    scratch = torch.empty(words // 4, dtype=torch.float32, device=dev) if words else None
    at = lambda t, items: None if t is None else t.data_ptr() + items * t.element_size()
    stat = rstd.contiguous()
    # More gains than a call takes go in parts of about one size, each with enough of them to need no scratch.
    most = -(-g.count // -(-g.count // _GRAD_GAINS)) if n else 1
    with _OnDevice(h):
        for i in range(0, g.count if n else 0, most):
            each = n // g.count
            gains, row = min(most, g.count - i), i * each
            _call("odp_rms_norm_grad", _stream(h), dtype_code(dtype), dtype_code(h.dtype), g.dt,
                  at(rows, row * rows.stride(0)), rows.stride(0), at(stat, row), at(y2, row * y2.stride(0)), y2.stride(0),
                  at(h2, 0 if h2 is None else row * h2.stride(0)), 0 if h2 is None else h2.stride(0), gains * each, width,
                  at(g.held, i * g.pitch), g.pitch, gains, offset, at(scratch, 0), at(dx, row * width),
                  at(dr, row * width), at(dw, i * width))
    return dx if need_x else None, (dx if same else dr) if need_r else None, dw


class _NormGrad(torch.autograd.Function):
    """Gradients of the norm; per example under vmap, the gains' too."""

    generate_vmap_rule = False

    @staticmethod
    def forward(gy, gh, h, rstd, weight, dtype, offset, groups, need_x, need_r, need_w):
        return _gradients(gy, gh, h, rstd, weight, dtype, offset, groups, need_x, need_r, need_w)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("rms_norm has no second derivative here")

    @staticmethod
    def vmap(info, in_dims, gy, gh, h, rstd, weight, dtype, offset, groups, need_x, need_r, need_w):
        n = info.batch_size
        gy, gh, h, rstd = (None if t is None else front(t, d, n) for t, d in zip((gy, gh, h, rstd), in_dims))
        each = 1 if groups is None else groups
        if weight is not None:
            weight = _batched_gain(weight, in_dims[4], n, groups)
        dx, dr, dw = _NormGrad.apply(gy, gh, h, rstd, weight, dtype, offset, n * each, need_x, need_r, need_w)
        if need_w and groups is not None:
            dw = dw.unflatten(0, (n, groups))
        return (dx, dr, dw), (0 if need_x else None, 0 if need_r else None, 0 if need_w else None)


def _batched_gain(weight, d, n, groups):
    """The gains of n times as many groups of rows: the batch before the groups."""
    if d is not None:
        weight = weight.movedim(d, 0)
        return weight.flatten(0, 1) if weight.dim() == 3 else weight
    if weight.dim() == 1 and groups is None:
        return weight.unsqueeze(0).expand(n, -1)
    return (weight.unsqueeze(0).expand(n, *weight.shape).flatten(0, 1) if weight.dim() == 2
            else weight.unsqueeze(0).expand(n * groups, -1))


def _merge(n, dims, x, residual, weight):
    """The operands of a batch of n as those of one call."""
    x = front(x, dims[0], n)
    residual = None if residual is None else front(residual, dims[1], n)
    if weight is not None and (dims[2] is not None or weight.dim() == 2):
        weight = _batched_gain(weight, dims[2], n, weight.shape[0] if dims[2] is None else None)
    return x, residual, weight


class _Norm(torch.autograd.Function):
    """(y, the sum or None, 1 / sqrt(..)); merges the batch under vmap."""

    generate_vmap_rule = False

    @staticmethod
    def forward(x, residual, weight, eps, offset):
        return _forward(x, residual, weight, eps, offset, True)[:3]

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, residual, weight, _, ctx.offset = inputs
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(output[2])
        ctx.save_for_backward(x if residual is None else output[1], output[2], weight)
        ctx.dtype = x.dtype

    @staticmethod
    def backward(ctx, gy, gh, _):
        if gy is None and gh is None:
            return None, None, None, None, None
        h, rstd, weight = ctx.saved_tensors
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        groups = weight.shape[0] if weight is not None and weight.dim() == 2 else None
        dx, dr, dw = _NormGrad.apply(gy, gh, h, rstd, weight, ctx.dtype, ctx.offset, groups, need_x, need_r, need_w)
        return dx, dr, dw, None, None

    @staticmethod
    def vmap(info, in_dims, x, residual, weight, eps, offset):
        x, residual, weight = _merge(info.batch_size, in_dims, x, residual, weight)
        host = None if transformed() else _bound()
        if host is not None:
            y, rstd, *h = host.rms_norm_kept(x, residual, weight, eps, offset)
            h = h[0] if h else None
        else:
            y, h, rstd = _Norm.apply(x, residual, weight, eps, offset)
        return (y, h, rstd), (0, 0 if h is not None else None, 0)


def _check(name, x, weight, residual, eps):
    if not isinstance(x, torch.Tensor) or x.dtype not in _ROW_DTYPES:
        raise TypeError(f"{name} supports float32, bfloat16 and float16 rows, got "
                        f"{x.dtype if isinstance(x, torch.Tensor) else type(x).__name__}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _WIDE:
        raise ValueError(f"{name} takes rows of 1 to {_WIDE} values, got {tuple(x.shape)}")
    if weight is not None:
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
        if weight.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must be shaped {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"residual must be {x.dtype} or float32, got {residual.dtype}")
    if x.device.type != "cuda" or any(t is not None and t.device != x.device for t in (weight, residual)):
        raise RuntimeError(f"{name} runs on the GPU: its arguments must be CUDA tensors of one device")
    if not 0.0 <= eps <= _F32.max:  # the kernels take it in float32
        raise ValueError(f"eps must be 0 or more and finite in float32, got {eps}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             eps: float = 1e-6, unit_offset: bool = False):
    """``h / sqrt(mean(h^2) + eps) * weight`` of every row, h = x or ``x + residual``.

    ``x`` [..., width] in float32, bfloat16 or float16, width up to 32768;
    ``weight`` [width] (None: 1; 1 + weight with ``unit_offset``) and
    ``residual`` [..., width] in x's type or float32.  Without a residual the
    norm is returned, in x's type; with one (the norm, h): h is the sum as the
    residual's type holds it, and the norm is of that.  Squares and sums are
    float32 and each result is rounded once, so rows whose squares leave
    float32 (beyond 1.8e19) give 0, as torch's do.  The gain's gradient is
    summed in float32.  No second and no forward-mode derivatives.
    """
    _check("rms_norm", x, weight, residual, eps)
    offset = 1.0 if unit_offset and weight is not None else 0.0
    host = _bound()
    if host is not None:
        if not transformed():
            out = host.rms_norm(x, residual, weight, eps, offset)
        else:
            out = merged(lambda n, dims, *ts: host.rms_norm(*_merge(n, dims, *ts), eps, offset), x, residual, weight)
        if out is not None:
            return tuple(out) if residual is not None else out[0]
    y, h, _ = _Norm.apply(x, residual, weight, float(eps), offset)
    return y if residual is None else (y, h)


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
                       eps: float = 1e-6, unit_offset: bool = False, block: int | None = None):
    """``rms_norm`` in 8 bits: (q, scales), with a residual (q, scales, h).

    q [..., width] is float8_e4m3fn, the norm over its scale rounded to
    nearest-even from float32.  ``scales`` float32 [...], the largest magnitude
    of the row over 448, or with ``block=128`` [..., ceil(width / 128)], that of
    every 128 columns; at least the least normal float32, so a row of zeros has
    a finite one (where ``eps`` is above 0).  A row (or block) that holds a NaN is NaN.  Not
    differentiable: no input may require a gradient, unless gradients are off, or
    have a forward-mode tangent.
    """
    _check("rms_norm_quantized", x, weight, residual, eps)
    if block not in (None, BLOCK):
        raise ValueError(f"block must be None (a scale per row) or {BLOCK}, got {block}")
    if transformed():
        raise NotImplementedError("rms_norm_quantized does not run inside torch.func transforms or clipped_grad")
    given = [t for t in (x, weight, residual) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise RuntimeError("rms_norm_quantized has no gradient: call it under torch.no_grad()")
    offset = 1.0 if unit_offset and weight is not None else 0.0
    quant, host = 2 if block else 1, _bound()
    if host is not None:
        return tuple(host.rms_norm_quantized(x, residual, weight, eps, offset, quant))
    no_tangent("the norm operators", x, residual, weight)
    q, h, _, scales = _forward(x, residual, weight, float(eps), offset, False, quant)
    return (q, scales) if residual is None else (q, scales, h)


class RMSNorm(torch.nn.Module):
    """``rms_norm`` with a gain; ``forward(x)`` or ``forward(x, residual)``."""

    def __init__(self, width: int, eps: float = 1e-6, *, unit_offset: bool = False, device=None, dtype=None) -> None:
        super().__init__()
        self.eps, self.unit_offset = eps, unit_offset
        make = torch.zeros if unit_offset else torch.ones
        self.weight = torch.nn.Parameter(make(width, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return rms_norm(x, self.weight, residual=residual, eps=self.eps, unit_offset=self.unit_offset)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, eps={self.eps}" + (", unit_offset=True" if self.unit_offset else "")


def route_norms(model: torch.nn.Module, types=(torch.nn.RMSNorm,)) -> list[str]:
    """Make the model's norms of the given classes ``RMSNorm``; returns their names, of a shared one each.

    Any class does whose forward is ``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, with a 1-D
    ``weight`` and ``eps`` or ``variance_epsilon`` (Hugging Face's): the product is rounded once here, where some round
    before the gain too.  The modules change their class in place, so gains, hooks, modes and sharing stay as they are.
    Norms without a gain, over several dimensions or with a ``forward`` of the instance's own stay.
    """
    found = []
    for name, mod in model.named_modules(remove_duplicate=False):
        weight = getattr(mod, "weight", None)
        if type(mod) not in tuple(types) or weight is None or weight.dim() != 1:
            continue
        if type(mod) is RMSNorm or "forward" in vars(mod):
            continue
        eps = getattr(mod, "eps", None) if hasattr(mod, "eps") else mod.variance_epsilon
        found.append((name, mod, _F32.eps if eps is None else float(eps)))  # torch's, of the type that it computes in
    for _, mod, eps in found:
        mod.__class__ = RMSNorm
        mod.eps, mod.unit_offset = eps, False
    return [name for name, _, _ in found]


__all__ = ["BLOCK", "RMSNorm", "rms_norm", "rms_norm_quantized", "route_norms"]
