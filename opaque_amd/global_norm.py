"""The norm of a whole tree of gradients, and the tree scaled to keep below a bound.

``clip_by_global_norm`` is what stands between the noise and the update: a bound
on the step, by the norm of the noisy gradients themselves.  That is
post-processing, which costs no privacy; the per-example clipping that does is
``clipped_grad``'s.

The work runs in the HIP kernels of ``libopaque_dp.so`` on the current stream,
leaves of any number and type in two passes; there is no CPU route.
"""

from __future__ import annotations

import torch

from opaque_amd import _native as N
from opaque_amd.capture import transformed
from opaque_amd.engine import dtype_code
from opaque_amd.pytree import tree_flatten, tree_unflatten
from opaque_amd.types import ClippedPytree, NoisedPytree
from opaque_amd.vocabulary import _bound, _call, _OnDevice, _stream, no_tangent

_LEAF_DTYPES = (torch.float32, torch.bfloat16, torch.float16, torch.float64)


def _dense(t: torch.Tensor) -> bool:
    """Whether the strides leave no gap and no overlap."""
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _tree_norm(leaves: list[torch.Tensor], clip: bool, max_norm: float, wide: bool):
    dev = leaves[0].device
    src = [t if _dense(t) else t.contiguous() for t in (t.resolve_neg() for t in leaves)]
    out = [torch.empty_like(t) for t in src] if clip else []
    table = torch.zeros(len(src), N.TN_FIELDS, dtype=torch.int64)
    for i, t in enumerate(src):
        table[i] = torch.tensor([t.data_ptr(), out[i].data_ptr() if clip else 0, t.numel(), dtype_code(t.dtype)])
    norm = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=dev)
    work = torch.empty(int(N.load().odp_tree_norm_scratch(len(src))) // 8, dtype=torch.float64, device=dev)
    with _OnDevice(norm):
        _call("odp_tree_norm", _stream(norm), table.data_ptr(), len(src), int(clip), max_norm, int(wide),
              work.data_ptr(), norm.data_ptr())
    return out, norm


def _checked(name: str, tensors: list[torch.Tensor]) -> bool:
    """Whether a leaf is float64; every one has to be of a type and on the device that the kernels take."""
    first, wide = tensors[0].device, False
    for t in tensors:
        if t.dtype not in _LEAF_DTYPES:
            raise TypeError(f"{name} supports float32, bfloat16, float16 and float64 leaves, got {t.dtype}")
        if t.device != first or first.type != "cuda":
            raise RuntimeError(f"{name} runs on the GPU: its leaves must be CUDA tensors of one device")
        wide |= t.dtype == torch.float64
    return wide


def _run(name: str, grads, max_norm: float | None):
    """(the scaled tree or None, the norm)."""
    if transformed():
        raise NotImplementedError(f"{name} does not run inside torch.func transforms")
    clip, host = max_norm is not None, _bound()
    if type(grads) is dict and all(type(t) is torch.Tensor for t in grads.values()):
        # The usual tree of a step: no structure to walk (20 us for 50 leaves).
        tensors, td = list(grads.values()), None
    else:
        leaves, td = tree_flatten(grads)
        if any(isinstance(t, ClippedPytree) for t in leaves):
            raise TypeError(f"{name} takes one tree of tensors: pass each clipped or noised pytree by itself")
        places = [i for i, t in enumerate(leaves) if isinstance(t, torch.Tensor)]
        tensors = [leaves[i] for i in places]
    if not tensors:
        return grads if td is None else tree_unflatten(td, leaves), torch.zeros(())
    if host is not None:
        out, norm = host.tree_norm(tensors, clip, max_norm or 0.0, name)
    else:
        wide = _checked(name, tensors)
        no_tangent("the tree norm's operators", *tensors)
        with torch.no_grad():
            out, norm = _tree_norm([t.detach() for t in tensors], clip, max_norm or 0.0, wide)
    if not clip:
        return None, norm
    if td is None:
        return dict(zip(grads, out)), norm
    for i, t in zip(places, out):
        leaves[i] = t
    return tree_unflatten(td, leaves), norm


def global_norm(tree) -> torch.Tensor:
    """The square root of the sum of all leaves' squares, a scalar tensor on their device.

    Leaves are float32, bfloat16, float16 or float64 CUDA tensors (others of the
    tree are passed over); squares and sums are float64 (those of float64 leaves
    also where their squares leave it) and the result float32, with a float64
    leaf float64.  Nothing is copied to the host, and the result has no gradient
    (a forward-mode tangent is an error).  An empty tree's norm is 0, on the CPU.
    """
    return _run("global_norm", tree.pytree if isinstance(tree, ClippedPytree) else tree, None)[1]


def clip_by_global_norm(grads, max_norm: float):
    """(the tree times ``min(1, max_norm / norm)``, its norm before): the norm over all leaves together.

    ``grads`` is a pytree of CUDA tensors as in ``global_norm``, or the
    ``NoisedPytree`` of a noise mechanism, of which the clipped leaves come back
    as a plain pytree: its ``noise_stddev`` no longer describes them.  A
    ``ClippedPytree`` is refused: its noise has to be added first.  Leaves keep
    their types and strides and are new tensors (one buffer per type); below the
    bound they are exact copies.  A NaN norm makes every entry NaN, an infinite
    one the finite entries 0.  The factor and the products are float32, float64
    for float64 leaves, and rounded once to the leaf's type.
    """
    if isinstance(grads, ClippedPytree):
        if not isinstance(grads, NoisedPytree):
            raise TypeError("clip_by_global_norm is post-processing: add the noise to a ClippedPytree first, or pass "
                            "its .pytree for gradients that stay private")
        grads = grads.pytree
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be 0 or more, got {max_norm}")
    return _run("clip_by_global_norm", grads, max_norm)


__all__ = ["clip_by_global_norm", "global_norm"]
