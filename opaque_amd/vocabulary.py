"""The two vocabulary ends of a language model: token embeddings and the loss over the vocabulary.

``embedding`` looks rows of a table up; its gradient adds the rows that come
back token by token, from positions sorted on the GPU.  Inside
``clipped_grad`` a table reached only through ``embedding`` (or the
``Embedding`` module) is a seam like the linear layers': the plan computes
every example's norm and the clipped sum from the tokens and the output
gradients, where ``vmap(grad)`` would make a dense [examples, vocabulary,
width] gradient (opaque-engine/.../clipping/_clipped_fun.py:756-762).

The work runs in the HIP kernels of ``libopaque_dp.so`` on the current
stream; there is no CPU route.
"""

from __future__ import annotations

import math

import torch

from opaque_amd import _native as N
from opaque_amd.capture import SiteRecord, active_session
from opaque_amd.engine import dtype_code

_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def pitched_rows(t: torch.Tensor) -> torch.Tensor:
    """2-D view [rows, d] with unit column stride and a pitch of at least d;
    rows laid out otherwise (transposed, expanded) are copied."""
    t2 = t.reshape(-1, t.shape[-1])
    if (t2.stride(1) != 1 and t2.shape[1] > 1) or t2.stride(0) < t2.shape[1]:
        t2 = t2.clone(memory_format=torch.contiguous_format)
    return t2


def _flat_tokens(tokens: torch.Tensor) -> torch.Tensor:
    return tokens.reshape(-1).contiguous()


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------


def _embed_rows(tokens: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    w = pitched_rows(weight.detach())
    flat = _flat_tokens(tokens)
    out = torch.empty((*tokens.shape, weight.shape[1]), dtype=weight.dtype, device=weight.device)
    if out.numel():
        with torch.cuda.device(weight.device):
            N.call("odp_embed_rows", _stream(weight), dtype_code(w.dtype), flat.data_ptr(), flat.element_size(),
                   flat.numel(), w.data_ptr(), w.stride(0), w.shape[0], w.shape[1], scale, out.data_ptr())
    return out


def table_gradient(tokens: torch.Tensor, g: torch.Tensor, vocab: int, scale: float, padding: int) -> torch.Tensor:
    """[vocab, width] = scale times the sum of each token's rows of g (the backward of ``embedding``)."""
    rows = pitched_rows(g.detach())
    flat = _flat_tokens(tokens)
    n, width, dev = flat.numel(), g.shape[-1], g.device
    out = torch.empty((vocab, width), dtype=g.dtype, device=dev)
    lib, dt = N.load(), dtype_code(g.dtype)
    sort = int(lib.odp_token_sort_scratch(n, vocab))
    words = max(sort, int(lib.odp_embed_sum_scratch(dt, n, width, 0))) // 4
    ids = torch.empty((2, n), dtype=torch.int32, device=dev)
    scratch = torch.empty(words, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        s = _stream(g)
        N.call("odp_token_sort", s, flat.data_ptr(), flat.element_size(), n, vocab, padding, None, None, 0,
               scratch.data_ptr(), ids[0].data_ptr(), ids[1].data_ptr(), None)
        N.call("odp_embed_grad", s, dt, rows.data_ptr(), rows.stride(0), n, width, ids[0].data_ptr(),
               ids[1].data_ptr(), vocab, scale, scratch.data_ptr(), out.data_ptr())
    return out


def _front(t: torch.Tensor, d: int | None, size: int) -> torch.Tensor:
    """The vmapped axis first (a shared tensor is expanded)."""
    return t.unsqueeze(0).expand(size, *t.shape) if d is None else t.movedim(d, 0)


class _EmbedGrad(torch.autograd.Function):
    """The table's gradient; per example under vmap."""

    generate_vmap_rule = False

    @staticmethod
    def forward(tokens, g, vocab, scale, padding):
        return table_gradient(tokens, g, vocab, scale, padding)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("embedding has no second derivative here")

    @staticmethod
    def vmap(info, in_dims, tokens, g, vocab, scale, padding):
        n = info.batch_size
        tokens, g = _front(tokens, in_dims[0], n), _front(g, in_dims[1], n)
        return torch.stack([_EmbedGrad.apply(tokens[i], g[i], vocab, scale, padding) for i in range(n)]), 0


class _Embed(torch.autograd.Function):
    """scale * weight[tokens]; merges the batch under vmap and, in a capture
    pass, records the tokens and the output gradient of an eligible table."""

    generate_vmap_rule = False

    @staticmethod
    def forward(tokens, weight, scale, padding):
        return _embed_rows(tokens, weight, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        tokens, weight, ctx.scale, ctx.padding = inputs
        ctx.save_for_backward(tokens)
        ctx.vocab = weight.shape[0]

    @staticmethod
    def backward(ctx, g):
        (tokens,) = ctx.saved_tensors
        dw = _EmbedGrad.apply(tokens, g, ctx.vocab, ctx.scale, ctx.padding) if ctx.needs_input_grad[1] else None
        return None, dw, None, None

    @staticmethod
    def vmap(info, in_dims, tokens, weight, scale, padding):
        n = info.batch_size
        tokens = _front(tokens, in_dims[0], n)
        if in_dims[1] is not None:  # a table per example (vmap(grad) over an expanded table)
            weight = weight.movedim(in_dims[1], 0)
            return torch.stack([_Embed.apply(tokens[i], weight[i], scale, padding) for i in range(n)]), 0
        sess = active_session()
        if sess is None or sess.mode != "capture" or id(weight) not in sess.eligible:
            return _Embed.apply(tokens, weight, scale, padding), 0
        rec = SiteRecord(x=None, A=None, B=None, scaling=scale, a_obj=None, b_obj=None, a_transposed=False,
                         b_transposed=False, w_obj=weight, tokens=tokens, padding=padding)
        sess.sites.append(rec)
        return _TapEmbed.apply(tokens, weight, scale, sess.anchor, rec), 0


class _TapEmbed(torch.autograd.Function):
    """Physical lookup that records the output gradient."""

    @staticmethod
    def forward(tokens, weight, scale, anchor, record):
        return _embed_rows(tokens, weight, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.record = inputs[4]

    @staticmethod
    def backward(ctx, g):
        ctx.record.g = g.detach()
        return None, None, None, torch.zeros((), dtype=torch.float32, device=g.device), None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[tokens]``: [*tokens.shape, width] in the table's dtype.

    ``weight`` [vocabulary, width] in float32, bfloat16 or float16, ``tokens``
    int64 or int32.  The product is rounded once; the gradient of the table
    is summed in float32 and rounded once.  A token outside the table gives a
    row of NaN and has no gradient; the table's row ``padding_idx`` is read
    but gets no gradient.
    """
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError("embedding tokens must be an int64 or int32 tensor")
    if weight.dim() != 2:
        raise ValueError(f"embedding weight must be [vocabulary, width], got {tuple(weight.shape)}")
    if weight.dtype not in _ROW_DTYPES:
        raise TypeError(f"embedding supports float32, bfloat16 and float16 tables, got {weight.dtype}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("embedding weight must not be empty")
    if weight.device.type != "cuda" or tokens.device != weight.device:
        raise RuntimeError("embedding runs on the GPU: tokens and weight must be CUDA tensors of one device")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    padding = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} outside the table of {weight.shape[0]} rows")
        padding = padding_idx % weight.shape[0]
    sess = active_session()
    if sess is not None and sess.mode == "discover":
        sess.uses[id(weight)] = sess.uses.get(id(weight), 0) + 1
        return _Embed.apply(tokens, weight.detach(), float(scale), padding)
    return _Embed.apply(tokens, weight, float(scale), padding)


class Embedding(torch.nn.Embedding):
    """``torch.nn.Embedding`` through ``embedding``, with a scale on its output."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, *,
                 scale: float = 1.0, device=None, dtype=None) -> None:
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = scale

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.weight, scale=self.scale, padding_idx=self.padding_idx)


__all__ = ["Embedding", "embedding"]
