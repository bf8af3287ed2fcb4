"""Routing of tokens to experts: what ``capture.moe`` takes as its index and weights.

``route`` turns a router's logits into the experts of every token and their
weights, in one launch, and the weights' gradient into the logits'; ``Router``
holds the router's weight, which is a full-weight seam under ``clipped_grad``.

The work runs in the HIP kernels of ``libopaque_dp.so`` on the current stream;
there is no CPU route.
"""

from __future__ import annotations

import math

import torch

from opaque_amd._vmap import front, merged
from opaque_amd.capture import Linear, transformed
from opaque_amd.engine import dtype_code
from opaque_amd.vocabulary import _F32, _bound, _call, _OnDevice, _stream, pitched_rows

_LOGIT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_EXPERTS, _CHOICES, _GROUPS = 1024, 64, 64  # ODP_ROUTE_EXPERTS, ODP_ROUTE_CHOICES
_SCORES = ("softmax", "sigmoid")
_BEST = ("top2", "max")


def _choose(z, bias, sigmoid, groups, top_groups, best, top_k, renorm, scale):
    rows = pitched_rows(z.detach())
    b = None if bias is None else bias.detach().resolve_neg().contiguous()
    shape = (*z.shape[:-1], top_k)
    index = torch.empty(shape, dtype=torch.int64, device=z.device)
    weights = torch.empty(shape, dtype=torch.float32, device=z.device)
    with _OnDevice(z):
        _call("odp_route", _stream(z), dtype_code(z.dtype), rows.data_ptr(), rows.stride(0), rows.shape[0],
              rows.shape[1], int(sigmoid), None if b is None else b.data_ptr(),
              b.shape[0] if b is not None and b.dim() == 2 else 1, groups, top_groups, best, top_k, int(renorm), scale,
              index.data_ptr(), weights.data_ptr())
    return index, weights


def _gradient(gw, z, index, sigmoid, top_k, renorm, scale):
    for t in (z, index):
        if t.device != gw.device:
            raise RuntimeError(f"routing operator: a saved tensor came back on {t.device}, not {gw.device}")
    if index.dtype != torch.int64 or index.shape != gw.shape or z.shape[:-1] != gw.shape[:-1]:
        raise RuntimeError("routing operator: a saved tensor came back otherwise than it was saved")
    rows, g, idx = pitched_rows(z.detach()), gw.detach().resolve_neg().contiguous(), index.contiguous()
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    with _OnDevice(z):
        _call("odp_route_grad", _stream(z), dtype_code(z.dtype), rows.data_ptr(), rows.stride(0), rows.shape[0],
              rows.shape[1], int(sigmoid), top_k, int(renorm), scale, idx.data_ptr(), g.data_ptr(), top_k,
              dz.data_ptr())
    return dz


class _RouteGrad(torch.autograd.Function):
    """The logits' gradient; merges the batch under vmap."""

    generate_vmap_rule = False

    @staticmethod
    def forward(gw, z, index, sigmoid, top_k, renorm, scale):
        return _gradient(gw, z, index, sigmoid, top_k, renorm, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("route has no second derivative here")

    @staticmethod
    def vmap(info, in_dims, gw, z, index, *rest):
        gw, z, index = (front(t, d, info.batch_size) for t, d in zip((gw, z, index), in_dims))
        return _RouteGrad.apply(gw, z, index, *rest), 0


def _merge(n, dims, z, bias):
    """The operands of a batch of n as those of one call."""
    z = front(z, dims[0], n)
    if bias is not None and (dims[1] is not None or bias.dim() == 2):
        # A bias per example; below another vmap the batch comes before its groups.
        bias = front(bias, dims[1], n)
        bias = bias.flatten(0, 1) if bias.dim() == 3 else bias
    return z, bias


class _Route(torch.autograd.Function):
    """(index, weights); merges the batch under vmap."""

    generate_vmap_rule = False

    @staticmethod
    def forward(z, bias, sigmoid, groups, top_groups, best, top_k, renorm, scale):
        return _choose(z, bias, sigmoid, groups, top_groups, best, top_k, renorm, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        z, _, ctx.sigmoid, _, _, _, ctx.top_k, ctx.renorm, ctx.scale = inputs
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(output[0])
        ctx.save_for_backward(z, output[0])

    @staticmethod
    def backward(ctx, _, gw):
        if gw is None or not ctx.needs_input_grad[0]:
            return (None,) * 9
        z, index = ctx.saved_tensors
        return _RouteGrad.apply(gw, z, index, ctx.sigmoid, ctx.top_k, ctx.renorm, ctx.scale), *(None,) * 8

    @staticmethod
    def vmap(info, in_dims, z, bias, *rest):
        z, bias = _merge(info.batch_size, in_dims, z, bias)
        host = None if transformed() else _bound()
        if host is not None:
            sigmoid, groups, top_groups, best, top_k, renorm, scale = rest
            return host.route(z, bias, sigmoid, groups, top_groups, best, top_k, renorm, scale), (0, 0)
        return _Route.apply(z, bias, *rest), (0, 0)


def route(logits: torch.Tensor, top_k: int, *, scores: str = "softmax", bias: torch.Tensor | None = None,
          groups: int = 1, top_groups: int = 1, group_best: str = "top2", renormalize: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``top_k`` experts of every token and their weights: (index int64, weights float32), both [..., top_k].

    ``logits`` [..., experts] in float32, bfloat16 or float16, up to 1024
    experts and 64 choices.  The scores are the experts' softmax or sigmoid;
    experts are ordered by score plus ``bias`` [experts] (float32; only the
    choice sees it, and it gets no gradient), best first.  With ``groups`` > 1
    (equal runs of experts, up to 64) only those of the ``top_groups`` best
    groups are open, by the sum of a group's two best or its best
    (``group_best`` "top2", "max").  Keys are compared as in 64 bits; equal ones
    go to the lower expert or group.  Without a bias, and without sums of groups
    where some stay shut, the logits themselves are compared, which order as the
    scores do and further apart.  The weights are ``scale`` times the chosen scores,
    over their sum with ``renormalize``; their gradient reaches the logits.

    An expert whose logit is -inf is masked: chosen after all others, with
    weight 0 (so is every expert of a row that is all masked).  A NaN, in a
    softmax also +inf, makes the row's weights NaN, for sigmoids those it takes
    part in.  The index holds different experts in any case.
    """
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _LOGIT_DTYPES:
        raise TypeError("route supports float32, bfloat16 and float16 logits, got "
                        f"{logits.dtype if isinstance(logits, torch.Tensor) else type(logits).__name__}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= _EXPERTS:
        raise ValueError(f"route takes logits of 1 to {_EXPERTS} experts, got {tuple(logits.shape)}")
    experts = logits.shape[-1]
    if scores not in _SCORES:
        raise ValueError(f"scores must be 'softmax' or 'sigmoid', got {scores!r}")
    if group_best not in _BEST:
        raise ValueError(f"group_best must be 'top2' or 'max', got {group_best!r}")
    if not 1 <= groups <= _GROUPS or experts % groups or not 1 <= top_groups <= groups:
        raise ValueError(f"{experts} experts do not make {groups} equal groups (1 to {_GROUPS}) with {top_groups} open")
    if not 1 <= top_k <= min(_CHOICES, experts // groups * top_groups):
        raise ValueError(f"top_k must be 1 to {min(_CHOICES, experts // groups * top_groups)}, got {top_k}")
    if bias is not None:
        if bias.shape != (experts,):
            raise ValueError(f"bias must be [{experts}], got {tuple(bias.shape)}")
        if bias.dtype != torch.float32:
            raise TypeError(f"bias must be float32, got {bias.dtype}")
    if logits.device.type != "cuda" or (bias is not None and bias.device != logits.device):
        raise RuntimeError("route runs on the GPU: its arguments must be CUDA tensors of one device")
    if not (math.isfinite(scale) and abs(scale) <= _F32.max):
        raise ValueError(f"scale must be finite in float32, got {scale}")
    bias = None if bias is None else bias.detach()
    args = (scores == "sigmoid", groups, top_groups, _BEST.index(group_best), top_k, bool(renormalize), float(scale))
    host = _bound()
    if host is not None:
        if not transformed():
            return host.route(logits, bias, *args)
        out = merged(lambda n, dims, z, b: host.route(*_merge(n, dims, z, b), *args), logits, bias)
        if out is not None:
            return out
    return _Route.apply(logits, bias, *args)


class Router(Linear):
    """A router: logits from its weight [experts, width], through the full-weight seam, then ``route``.

    ``balance=True`` registers a float32 buffer ``balance`` [experts] of zeros that a training
    loop may move against the experts' load; it stays float32 where the module is cast, as its
    steps are small.  ``forward`` returns (index, weights) for ``capture.moe``.
    """

    def __init__(self, width: int, experts: int, top_k: int, *, scores: str = "softmax", balance: bool = False,
                 groups: int = 1, top_groups: int = 1, group_best: str = "top2", renormalize: bool = True,
                 scale: float = 1.0, device=None, dtype=None) -> None:
        super().__init__(width, experts, bias=False, device=device, dtype=dtype)
        self.top_k = top_k
        self.options = {"scores": scores, "groups": groups, "top_groups": top_groups, "group_best": group_best,
                        "renormalize": renormalize, "scale": scale}
        self.register_buffer("balance", torch.zeros(experts, dtype=torch.float32, device=device) if balance else None)

    def _apply(self, fn, recurse=True):
        kept = self.balance
        super()._apply(fn, recurse)
        if kept is not None and self.balance.dtype != torch.float32:
            self.balance = kept.to(self.balance.device, torch.float32)
        return self

    def forward(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        bias = None if self.balance is None else self.balance.float()  # a caller may bring another buffer
        return route(super().forward(x), self.top_k, bias=bias, **self.options)


__all__ = ["Router", "route"]
