"""Below one vmap level without a rule's way there.

An autograd.Function under ``torch.func.vmap`` costs 115 us of host time for its
rule's dispatch (operands flattened, wrapped and unwrapped, outputs compared).
Where one vmap is the only transform that is active, as in the capture pass of
``clipped_grad``, the operators whose rule merges the batch take their operands
out of it, make the merged call, and put the results back, for 22.
"""

from __future__ import annotations

from collections.abc import Callable

import torch

_F = torch._C._functorch
_VMAP = _F.TransformType.Vmap


def front(t: torch.Tensor, d: int | None, size: int) -> torch.Tensor:
    """The batch first (a shared tensor is expanded)."""
    return t.unsqueeze(0).expand(size, *t.shape) if d is None else t if d == 0 else t.movedim(d, 0)


def merged(call: Callable, *operands: torch.Tensor | None):
    """``call(size, dims, *physical operands)`` below the one active vmap, its outputs batched in front; None where
    another transform is active or no operand is batched.  ``dims``: each operand's batch dimension or None."""
    top = _F.peek_interpreter_stack()
    level = 0 if top is None else top.level()
    if level != 1 or top.key() != _VMAP:  # levels count from 1
        return None
    values, dims, size = [], [], None
    for t in operands:
        if t is not None and _F.is_batchedtensor(t):
            dims.append(_F.maybe_get_bdim(t))
            t = _F.get_unwrapped(t)
            size = t.shape[dims[-1]]
        else:
            dims.append(None)
        values.append(t)
    if size is None:
        return None
    layer = _F.pop_dynamic_layer_stack()
    try:
        out = call(size, dims, *values)
    finally:
        _F.push_dynamic_layer_stack(layer)
    return tuple(_F._add_batch_dim(t, 0, level) for t in out)


__all__ = ["front", "merged"]
