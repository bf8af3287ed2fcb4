"""The two vocabulary ends of a language model: token embeddings and the loss over the vocabulary.

``embedding`` looks rows of a table up; its gradient adds the rows that come
back token by token, from positions sorted on the GPU.  Inside
``clipped_grad`` a table reached only through ``embedding`` (or the
``Embedding`` module) is a seam like the linear layers': the plan computes
every example's norm and the clipped sum from the tokens and the output
gradients, where ``vmap(grad)`` would make a dense [examples, vocabulary,
width] gradient (opaque-engine/.../clipping/_clipped_fun.py:756-762).

The work runs in the HIP kernels of ``libopaque_dp.so`` on the current
stream; there is no CPU route.  Outside torch.func the host helper makes the
calls; inside it (and without the helper) the Functions below do, whose vmap
rules merge the batch.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from opaque_amd import _host
from opaque_amd import _native as N
from opaque_amd.capture import SiteRecord, active_session, transformed
from opaque_amd.engine import dtype_code

_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_F32 = torch.finfo(torch.float32)


_functions: dict[str, object] = {}


def _call(name: str, *args) -> None:
    """A C entry point through a kept handle (these calls are a few microseconds of host time)."""
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(N.load(), name)
    rc = f(*args)
    if rc != N.ODP_OK:
        N.check(rc, name)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


class _OnDevice:
    """Makes a tensor's device current where it is not."""

    def __init__(self, t: torch.Tensor) -> None:
        self.ctx = None if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self) -> None:
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc) -> None:
        if self.ctx is not None:
            self.ctx.__exit__(*exc)


_host_ready: list = []


def _bound():
    """The host helper with the library's entry points bound, or None when it has not been built."""
    if not _host_ready:
        host, lib = _host.load(), N.load()
        if host is not None:
            at = {name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in N.exported_symbols()}
            host.bind(at)
            host.bind_block(at)
        _host_ready.append(host)
    return _host_ready[0]


def _on_one_device(t: torch.Tensor, *saved: torch.Tensor) -> None:
    """What comes back from autograd lies where the gradient does, wherever its hooks had it meanwhile."""
    for s in saved:
        if s.device != t.device:
            raise RuntimeError(f"vocabulary operators: a saved tensor came back on {s.device}, not {t.device}")


def no_tangent(who: str, *tensors: torch.Tensor | None) -> None:
    """A forward-mode tangent would be dropped without a word where no autograd.Function takes the call."""
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{who} have no forward-mode derivative")


def pitched_rows(t: torch.Tensor) -> torch.Tensor:
    """2-D view [rows, d] with unit column stride and a pitch of at least d;
    rows laid out otherwise (transposed, expanded) are copied."""
    t = t.resolve_neg()
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if (t2.stride(1) != 1 and t2.shape[1] > 1) or t2.stride(0) < t2.shape[1]:
        t2 = t2.clone(memory_format=torch.contiguous_format)
    return t2


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------


@functools.lru_cache(maxsize=256)
def _grad_words(dt: int, n: int, vocab: int, width: int) -> int:
    """float32 words of scratch of a table gradient: the sort's, then the sums'."""
    lib = N.load()
    return max(int(lib.odp_token_sort_scratch(n, vocab)), int(lib.odp_embed_sum_scratch(dt, n, width, 0))) // 4


def _embed_rows(tokens: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    w = pitched_rows(weight.detach())
    flat = tokens.contiguous()
    vocab, width = weight.shape
    out = torch.empty((*tokens.shape, width), dtype=weight.dtype, device=weight.device)
    n = flat.numel()
    if n:
        with _OnDevice(weight):
            _call("odp_embed_rows", _stream(weight), dtype_code(w.dtype), flat.data_ptr(), flat.element_size(), n,
                  w.data_ptr(), w.stride(0), vocab, width, scale, out.data_ptr())
    return out


def table_gradient(tokens: torch.Tensor, g: torch.Tensor, vocab: int, scale: float, padding: int) -> torch.Tensor:
    """[vocab, width] = scale times the sum of each token's rows of g (the backward of ``embedding``)."""
    rows = pitched_rows(g.detach())
    flat = tokens.contiguous()
    _on_one_device(g, tokens)
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.numel() != rows.shape[0]:
        raise RuntimeError("vocabulary operators: the saved tokens came back otherwise than they were saved")
    n, width, dev = flat.numel(), g.shape[-1], g.device
    dt = dtype_code(g.dtype)
    out = torch.empty((vocab, width), dtype=g.dtype, device=dev)
    words = (_grad_words(dt, n, vocab, width) + 3) // 4 * 4
    scratch = torch.empty(words + 2 * n, dtype=torch.int32, device=dev)
    at = scratch.data_ptr()
    keys = at + 4 * words
    with _OnDevice(g):
        s = _stream(g)
        _call("odp_token_sort", s, flat.data_ptr(), flat.element_size(), n, vocab, padding, None, None, 0, at, keys,
              keys + 4 * n, None, out.data_ptr(), out.numel() * out.element_size())
        _call("odp_embed_grad", s, dt, rows.data_ptr(), rows.stride(0), n, width, keys, keys + 4 * n, vocab, scale, at,
              out.data_ptr())
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
        if sess is None or sess.mode != "capture" or id(weight) not in sess.eligible or transformed():
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
    if not abs(scale) <= _F32.max:  # the kernels take it in float32
        raise ValueError(f"scale must be finite in float32, got {scale}")
    padding = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} outside the table of {weight.shape[0]} rows")
        padding = padding_idx % weight.shape[0]
    sess = active_session()
    if sess is not None and sess.mode == "discover":
        weight = sess.hide(weight)
    elif sess is not None and id(weight) in sess.eligible:
        tokens = sess.batched(tokens)
    host = None if transformed() else _bound()
    if host is not None:
        return host.embedding(tokens, weight, scale, padding)
    return _Embed.apply(tokens, weight, float(scale), padding)


class Embedding(torch.nn.Embedding):
    """``torch.nn.Embedding`` through ``embedding``, with a scale on its output."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, *,
                 scale: float = 1.0, device=None, dtype=None) -> None:
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: int | None = None, *,
                        scale: float = 1.0) -> Embedding:
        """A module on a given table (shared, not copied), frozen unless told otherwise."""
        if embeddings.dim() != 2:
            raise ValueError(f"embeddings must be [vocabulary, width], got {tuple(embeddings.shape)}")
        m = cls(*embeddings.shape, padding_idx, scale=scale, device="meta", dtype=embeddings.dtype)
        m.weight = torch.nn.Parameter(embeddings, requires_grad=not freeze)
        return m

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.weight, scale=self.scale, padding_idx=self.padding_idx)


# ---------------------------------------------------------------------------
# Linear cross entropy
# ---------------------------------------------------------------------------

_HEAD_DTYPES = (torch.float32, torch.bfloat16)
# Bytes of d (the logits' gradient, in the inputs' type) that the backward
# holds at a time: a piece of the vocabulary for all tokens.
PIECE_BYTES = 512 << 20
_PIECE_COLUMNS = 1 << 22  # a piece's columns stay below it (ODP_XENT_PIECE)
_WIDE = 1 << 20  # rows of the head are narrower and less far apart (ODP_XENT_WIDE)
_STAT = 3  # float32 words that the forward leaves of a row for the backward (ODP_XENT_STAT)
# Bytes of float32 logits up to which the process's live losses together (1.5 %
# of the memory of one GPU) keep them for their backward passes, where that is
# faster than forming them again; 0 keeps none.  Neither do the gradients of torch.func
# (``vmap(grad)``) and of a head that trains under ``clipped_grad``.
KEEP_BYTES = 4 << 30
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _lanes(dtype: torch.dtype) -> int:
    """Elements in 16 bytes."""
    return 4 if dtype == torch.float32 else 8


def _head_rows(weight: torch.Tensor) -> torch.Tensor:
    """The head with rows on the 16-byte grid, less than ODP_XENT_WIDE apart: itself, or a copy whose width is padded
    with zeros."""
    w, per = pitched_rows(weight.detach()), _lanes(weight.dtype)
    if w.shape[1] % per == 0 and w.stride(0) % per == 0 and w.stride(0) < _WIDE and w.data_ptr() % 16 == 0:
        return w
    wide = w.new_zeros(w.shape[0], -(-w.shape[1] // per) * per)
    wide[:, : w.shape[1]] = w
    return wide


@functools.lru_cache(maxsize=256)
def _xent_words(dt: int, n: int, width: int, vocab: int) -> tuple[int, int]:
    """float32 words of the statistics' scratch and of dx's sums."""
    lib = N.load()
    return (max(int(lib.odp_xent_stats_scratch(dt, n, vocab)) // 4, 1),
            max(int(lib.odp_xent_dx_scratch(dt, n, width)) // 4, 1))


@functools.lru_cache(maxsize=256)
def _dw_words(dt: int, n: int, vc: int, width: int) -> int:
    """float32 words that the slices of the tokens of a piece of dW take (0: not split)."""
    return int(N.load().odp_xent_dw_scratch(dt, n, vc, width)) // 4


@functools.lru_cache(maxsize=256)
def _xent_pitch(dt: int, columns: int) -> int:
    return int(N.load().odp_xent_pitch(dt, columns))


class _Packed:
    """The rows that bear a loss, gathered (every row with ``keep``)."""

    def __init__(self, x: torch.Tensor, w: torch.Tensor, target: torch.Tensor, ignore: int, keep: bool = False,
                 losses: torch.Tensor | None = None, stat: torch.Tensor | None = None) -> None:
        rows, flat = pitched_rows(x.detach()), target.contiguous()
        self.dt, self.n, self.cols = dtype_code(x.dtype), flat.numel(), rows.shape[1]
        self.w, self.vocab, self.width = w, w.shape[0], w.shape[1]
        dev, room = x.device, max(self.n, 1)
        self.xc = torch.empty((room, self.width), dtype=x.dtype, device=dev)
        self.ids = torch.empty(3 * room + 2, dtype=torch.int32, device=dev)
        at = self.ids.data_ptr()
        self.count = at
        self.act, self.tgt, self.where = (at + 8 + 4 * k * room for k in range(3))
        _call("odp_xent_rows", _stream(x), self.dt, rows.data_ptr(), rows.stride(0), self.n, self.cols, self.width,
              flat.data_ptr(), flat.element_size(), self.vocab, ignore, int(keep), self.xc.data_ptr(), self.act,
              self.tgt, self.where, self.count, None if losses is None else losses.data_ptr(),
              None if stat is None else stat.data_ptr())

    def losses(self, softcap: float, losses: torch.Tensor, stat: torch.Tensor) -> None:
        scratch = torch.empty(_xent_words(self.dt, self.n, self.width, self.vocab)[0], dtype=torch.float32,
                              device=self.xc.device)
        _call("odp_xent_losses", _stream(self.xc), self.dt, self.xc.data_ptr(), self.n, self.width, self.act,
              self.tgt, self.count, self.w.data_ptr(), self.w.stride(0), self.vocab, softcap, scratch.data_ptr(),
              losses.data_ptr(), stat.data_ptr(), None, 0)

    def piece(self, whole: bool = False) -> int:
        """Columns of the vocabulary a piece of d holds: as many pieces as PIECE_BYTES makes, of one size."""
        edge = _xent_pitch(self.dt, 1)
        fit = max(min(PIECE_BYTES // (max(self.n, 1) * self.xc.element_size()) // edge * edge, _PIECE_COLUMNS - edge),
                  edge)
        pieces = -(-self.vocab // fit)
        return self.vocab if whole else min(self.vocab, -(-(-(-self.vocab // pieces)) // edge) * edge)

    def gradients(self, softcap: float, stat: torch.Tensor, g: torch.Tensor, x_shape: torch.Size | None,
                  need_w: bool, keep_d: bool = False):
        """(dx, dW, d): dx where ``x_shape`` is given; d [n, vocab] where
        ``keep_d`` (packed with ``keep``).  ``g`` holds one gradient per row."""
        dev, dtype, dt = self.xc.device, self.xc.dtype, self.dt
        piece = self.piece(keep_d)
        d = torch.empty((max(self.n, 1), _xent_pitch(dt, piece)), dtype=dtype, device=dev)
        dx = dw = sums = None
        s = _stream(self.xc)
        if x_shape is not None:
            dx = torch.empty(x_shape, dtype=dtype, device=dev)
            sums = torch.empty(_xent_words(dt, self.n, self.width, self.vocab)[1], dtype=torch.float32, device=dev)
        if need_w:
            dw = torch.empty((self.vocab, self.width), dtype=dtype, device=dev)
        rest = torch.empty(max(self.n, 1), dtype=torch.float32, device=dev)
        w, ldw, xc = self.w.data_ptr(), self.w.stride(0), self.xc.data_ptr()
        for v0 in range(0, self.vocab, piece):
            vc = min(piece, self.vocab - v0)
            ldd = _xent_pitch(dt, vc)
            _call("odp_xent_dlogits", s, dt, xc, self.n, self.width, self.act, self.tgt, self.count, w, ldw,
                  self.vocab, softcap, v0, vc, stat.data_ptr(), g.data_ptr(), 1, None, None, 0, d.data_ptr(),
                  ldd, rest.data_ptr())
            if dx is not None:
                _call("odp_xent_dx", s, dt, self.n, self.width, self.count, w, ldw, self.vocab, v0, vc, piece,
                      d.data_ptr(), ldd, sums.data_ptr())
            if dw is not None:
                slots = torch.empty(_dw_words(dt, self.n, vc, self.width), dtype=torch.float32, device=dev)
                _call("odp_xent_dw", s, dt, xc, self.n, self.width, self.count, vc, d.data_ptr(), ldd,
                      slots.data_ptr(), dw.data_ptr() + v0 * self.width * dw.element_size(), self.width)
        if dx is not None:
            _call("odp_xent_dx_rows", s, dt, self.n, self.cols, self.width, self.count, self.where, self.tgt, w,
                  ldw, piece, sums.data_ptr(), rest.data_ptr(), dx.data_ptr())
        if dw is not None and self.cols != self.width:
            dw = dw[:, : self.cols].contiguous()
        return dx, dw, d[: self.n, : self.vocab] if keep_d else None


def _xent_losses(x, weight, target, softcap, ignore):
    losses = torch.empty(target.shape, dtype=torch.float32, device=x.device)
    stat = torch.empty((*target.shape, _STAT), dtype=torch.float32, device=x.device)
    with _OnDevice(x):
        p = _Packed(x, _head_rows(weight), target, ignore, False, losses, stat)
        p.losses(softcap, losses, stat)
    return losses, stat


def _xent_gradients(g, x, weight, target, stat, softcap, ignore, need_x, need_w, keep_d=False):
    g, stat = g.detach().float().contiguous().reshape(-1), stat.contiguous()
    _on_one_device(g, x, weight, target, stat)
    n = g.numel()
    if (x.dtype != weight.dtype or x.shape[-1] != weight.shape[1] or stat.dtype != torch.float32
            or (target.numel(), stat.numel(), x.numel()) != (n, n * _STAT, n * x.shape[-1])):
        raise RuntimeError("vocabulary operators: a saved tensor came back otherwise than it was saved")
    with _OnDevice(x):
        p = _Packed(x, _head_rows(weight), target, ignore, keep_d)
        return p.gradients(softcap, stat, g, x.shape if need_x else None, need_w, keep_d)


class _XentGrad(torch.autograd.Function):
    """Gradients of the token losses; per example under vmap."""

    generate_vmap_rule = False

    @staticmethod
    def forward(g, x, weight, target, stat, softcap, ignore, need_x, need_w):
        dx, dw, _ = _xent_gradients(g, x, weight, target, stat, softcap, ignore, need_x, need_w)
        return dx, dw

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("linear_cross_entropy has no second derivative here")

    @staticmethod
    def vmap(info, in_dims, g, x, weight, target, stat, softcap, ignore, need_x, need_w):
        n = info.batch_size
        g, x, target, stat = (_front(t, d, n) for t, d in zip((g, x, target, stat), (*in_dims[:2], *in_dims[3:5])))
        if in_dims[2] is None and not need_w:  # one head: the batch is one set of rows
            return _XentGrad.apply(g, x, weight, target, stat, softcap, ignore, need_x, need_w), (0, None)
        w = _front(weight, in_dims[2], n)
        out = [_XentGrad.apply(g[i], x[i], w[i], target[i], stat[i], softcap, ignore, need_x, need_w)
               for i in range(n)]
        return (torch.stack([o[0] for o in out]) if need_x else None,
                torch.stack([o[1] for o in out]) if need_w else None), (0 if need_x else None, 0 if need_w else None)


class _Xent(torch.autograd.Function):
    """Token losses [*target.shape] and their rows' statistics; merges the batch
    under vmap and, in a capture pass, records x and the logits' gradient of
    an eligible head."""

    generate_vmap_rule = False

    @staticmethod
    def forward(x, weight, target, softcap, ignore):
        return _xent_losses(x, weight, target, softcap, ignore)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight, target, ctx.softcap, ctx.ignore = inputs
        ctx.mark_non_differentiable(output[1])
        ctx.save_for_backward(x, weight, target, output[1])

    @staticmethod
    def backward(ctx, g, _):
        x, weight, target, stat = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        dx, dw = _XentGrad.apply(g, x, weight, target, stat, ctx.softcap, ctx.ignore, need_x, need_w)
        return dx, dw, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, weight, target, softcap, ignore):
        n = info.batch_size
        x, target = _front(x, in_dims[0], n), _front(target, in_dims[2], n)
        if in_dims[1] is not None:  # a head per example
            w = weight.movedim(in_dims[1], 0)
            out = [_Xent.apply(x[i], w[i], target[i], softcap, ignore) for i in range(n)]
            return (torch.stack([o[0] for o in out]), torch.stack([o[1] for o in out])), (0, 0)
        sess = active_session()
        if sess is None or sess.mode != "capture" or id(weight) not in sess.eligible or transformed():
            host = None if transformed() else _bound()
            if host is not None:
                return host.token_losses(x, weight, target, softcap, ignore, PIECE_BYTES, KEEP_BYTES), (0, 0)
            return _Xent.apply(x, weight, target, softcap, ignore), (0, 0)
        rec = SiteRecord(x=x, A=None, B=None, scaling=1.0, a_obj=None, b_obj=None, a_transposed=False,
                         b_transposed=False, w_obj=weight)
        sess.sites.append(rec)
        return _TapXent.apply(x, weight, target, softcap, ignore, sess.anchor, rec), (0, 0)


class _TapXent(torch.autograd.Function):
    """Physical losses of a head that trains under ``clipped_grad``: the
    backward keeps d (the logits' gradient, [rows, vocabulary] in the
    inputs' type), from which the plan takes the head's per-example norms and
    clipped sum as of any full-weight linear."""

    @staticmethod
    def forward(x, weight, target, softcap, ignore, anchor, record):
        return _xent_losses(x, weight, target, softcap, ignore)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight, target, ctx.softcap, ctx.ignore, _, ctx.record = inputs
        ctx.mark_non_differentiable(output[1])
        ctx.save_for_backward(x, weight, target, output[1])

    @staticmethod
    def backward(ctx, g, _):
        x, weight, target, stat = ctx.saved_tensors
        dx, _, d = _xent_gradients(g, x, weight, target, stat, ctx.softcap, ctx.ignore, ctx.needs_input_grad[0],
                                   False, keep_d=True)
        ctx.record.g = d[: target.numel()].unflatten(0, target.shape) if target.dim() > 1 else d
        return dx, None, None, None, None, torch.zeros((), dtype=torch.float32, device=g.device), None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                         softcap: float | None = None, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``x weight^T`` against ``target``, a piece of the vocabulary at a time.

    ``x`` [..., width] and ``weight`` [vocabulary, width] are both float32 or
    both bfloat16, ``target`` [...] int64 or int32.  ``softcap`` bounds the
    logits as ``softcap * tanh(logits / softcap)``.  ``reduction`` "none"
    gives the float32 loss of every token, "sum" and "mean" their sum and
    mean over the tokens whose target is not ``ignore_index`` (NaN when there
    is none, as torch's).  A target outside the vocabulary makes its loss and
    its row of x's gradient NaN, and is left out of the head's.  Logits
    and statistics are float32; the gradients are summed in float32 and
    rounded once, from logit gradients in the inputs' type.  No [tokens,
    vocabulary] tensor is made beyond a piece of PIECE_BYTES in the backward
    and, where all live losses' take at most KEEP_BYTES, the logits between
    the passes.

    Replaces the reference's linear cross entropy
    (opaque-patches/.../kernels/linear_cross_entropy.py:249).  Inside
    ``clipped_grad`` a trainable head reached only through it is a seam.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"x [..., width] and weight [vocabulary, width] do not match: {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target must be shaped {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"target must be int64 or int32, got {target.dtype}")
    if x.dtype != weight.dtype or x.dtype not in _HEAD_DTYPES:
        raise TypeError(f"x and weight must both be float32 or both bfloat16, got {x.dtype} and {weight.dtype}")
    if weight.device.type != "cuda" or x.device != weight.device or target.device != weight.device:
        raise RuntimeError("linear_cross_entropy runs on the GPU: its arguments must be CUDA tensors of one device")
    if softcap is not None and not _F32.tiny <= softcap <= _F32.max:
        raise ValueError(f"softcap must be positive and finite (and normal in float32), got {softcap}")
    sess = active_session()
    if sess is not None and sess.mode == "discover":
        weight = sess.hide(weight)
    host = None if transformed() else _bound()
    if host is not None:
        return host.cross_entropy(x, weight, target, softcap or 0.0, ignore_index, _REDUCTIONS[reduction], PIECE_BYTES,
                                  KEEP_BYTES)
    losses, _ = _Xent.apply(x, weight, target, float(softcap or 0.0), int(ignore_index))
    if reduction == "none":
        return losses
    total = losses.double().sum().float()  # added in 64 bits and rounded once
    return total if reduction == "sum" else total / (target != ignore_index).sum()


__all__ = ["Embedding", "embedding", "linear_cross_entropy"]
