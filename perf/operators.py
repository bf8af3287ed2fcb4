"""The vocabulary operators as measurable cases.

A language model meets its vocabulary twice: the embedding turns tokens into
rows, the loss turns the last hidden rows into log-probabilities of the next
tokens.  ``kind`` names the operator:

  loss    linear_cross_entropy: softmax cross entropy of x W^T over the whole
          vocabulary; ``grad`` says which gradients the pass returns ("none",
          "x": the head is frozen as under LoRA, "xw": the head trains)
  lookup  embedding: rows of the table times a scale; with ``grad`` also the
          dense gradient of the table
  clip    the embedding's part of a DP step: per-example norms of the table's
          gradient, clip factors and the clipped sum, through GhostPlan

With ``own`` false every case runs as elementary torch operations in float32,
rounded once at the end.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100
GAMMA = 0.01  # AUTO-S


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _loss(name, **kw):
    return {"name": name, "kind": "loss", "dtype": "bf16", "tokens": 4096, "width": 4096, "vocab": 128256,
            "ignored": 0.0, "softcap": 0.0, "grad": "x", **kw}


def _lookup(name, **kw):
    return {"name": name, "kind": "lookup", "dtype": "bf16", "tokens": 4096, "width": 4096, "vocab": 128256,
            "scaled": False, "padded": 0.0, "grad": True, **kw}


def _clip(name, **kw):
    return {"name": name, "kind": "clip", "dtype": "bf16", "batch": 16, "seq": 1024, "width": 4096,
            "vocab": 128256, "padded": 0.0, **kw}


def listed():
    return [
        # The log-probability of one decoded token: the head read once.
        _loss("score_one", tokens=1, grad="none"),
        # The same for a batch of decoded sequences, a smaller model.
        _loss("score_batch", tokens=47, width=2048, vocab=32000, grad="none"),
        # LoRA in float32 on a GPT-2-sized model, 4 x 256 tokens, a frozen head.
        _loss("frozen_f32", dtype="f32", tokens=1024, width=768, vocab=50257),
        # LoRA fine-tuning on answers after prompts (whose tokens bear no loss), Llama-3-8B-shaped head.
        _loss("frozen_answers", tokens=5120, ignored=0.5),
        # Odd sizes with a softcap, every weight trained.
        _loss("train_odd", tokens=777, width=1000, vocab=32003, ignored=0.1, softcap=30.0, grad="xw"),
        # Full-weight training of the Llama-3-8B-shaped head: the largest.
        _loss("train_full", grad="xw"),
        # The embeddings of a batch of decoded tokens: latency.
        _lookup("decode", tokens=16, grad=False),
        # Odd width, small vocabulary, many repeats, half padding.
        _lookup("table_odd", dtype="f16", tokens=1023, width=321, vocab=1001, scaled=True, padded=0.5),
        # GPT-2-sized table in float32.
        _lookup("table_f32", dtype="f32", tokens=16384, width=768, vocab=50257),
        # A long batch on the Llama-3-8B-shaped table.
        _lookup("table_long", tokens=32768, scaled=True, padded=0.2),
        # DP step of a small table: 8 short examples.
        _clip("clip_short", dtype="f32", batch=8, seq=61, width=768, vocab=50257),
        # DP step of the Llama-3-8B-shaped table, examples padded to 1024 tokens.
        _clip("clip_train", padded=0.4),
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v // step * step))


def draw(rng):
    kind = rng.choice(["loss", "loss", "lookup", "clip"])
    if kind == "loss":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        width = _log_int(rng, 256, 4096 if dtype == "bf16" else 1536, 8)
        vocab = _log_int(rng, 1000, 131072)
        most = min(8192, 4096 * 4096 * 128256 // (width * vocab)) if dtype == "bf16" else 2048
        return {"kind": "loss", "dtype": dtype, "tokens": _log_int(rng, 1, most), "width": width, "vocab": vocab,
                "ignored": rng.choice([0.0, 0.3, 0.7]), "softcap": rng.choice([0.0, 0.0, 30.0]),
                "grad": rng.choice(["none", "x", "xw"])}
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"]) if kind == "lookup" else rng.choice(["bf16", "bf16", "f32"])
    width = _log_int(rng, 64, 4096)
    vocab = _log_int(rng, 500, 131072)
    if kind == "lookup":
        return {"kind": "lookup", "dtype": dtype, "tokens": _log_int(rng, 1, 32768), "width": width, "vocab": vocab,
                "scaled": rng.random() < 0.5, "padded": rng.choice([0.0, 0.2, 0.6]), "grad": rng.random() < 0.7}
    batch = _log_int(rng, 1, 64)
    return {"kind": "clip", "dtype": dtype, "batch": batch, "seq": _log_int(rng, 4, 16384 // batch), "width": width,
            "vocab": vocab, "padded": rng.choice([0.0, 0.2, 0.6])}


def _active(case):
    """Tokens that bear a loss."""
    return case["tokens"] - int(case["tokens"] * case["ignored"])


def work(case):
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    d, v = case["width"], case["vocab"]
    if case["kind"] == "loss":
        n, k = case["tokens"], _active(case)
        grads = {"none": 0, "x": 1, "xw": 2}[case["grad"]]
        return {"bytes": k * d * e + v * d * e + 8 * n + 4 * n + (n * d * e if grads else 0)
                + (v * d * e if grads == 2 else 0), "flops": 2.0 * k * v * d * (1 + grads)}
    if case["kind"] == "lookup":
        n = case["tokens"]
        return {"bytes": 8 * n + 2 * n * d * e + (n * d * e + v * d * e if case["grad"] else 0), "flops": 0}
    n = case["batch"] * case["seq"]
    return {"bytes": 8 * n + n * d * e + v * d * e + 4 * case["batch"], "flops": 0}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _tokens(g, n, vocab):
    """Token ids with the frequencies of text: the log of the id is uniform."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)


def _loss_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    n, d, v = case["tokens"], case["width"], case["vocab"]
    w = (torch.randn(v, d, generator=g, device=DEV) / math.sqrt(d)).to(dt)
    y = _tokens(g, n, v)
    # Hidden rows lean toward their target by up to what makes it likely, as
    # in a trained model: p(target) from 1 / vocab to near 1.
    lean = torch.rand(n, 1, generator=g, device=DEV) * 1.5 * math.log(v)
    x = (torch.randn(n, d, generator=g, device=DEV) + lean * w[y].float()).to(dt)
    # The first part of each of four examples bears no loss.
    off = n - _active(case)
    rank = torch.arange(n, device=DEV) * 4 % max(n, 1)
    y[torch.argsort(rank, stable=True)[:off]] = IGNORE
    return x, w, y


def _lookup_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    n, d, v = case["tokens"], case["width"], case["vocab"]
    w = (0.02 * torch.randn(v, d, generator=g, device=DEV)).to(dt)
    y = _tokens(g, n, v)
    y[n - int(n * case["padded"]):] = v // 2  # one padding token, an ordinary row of the table
    go = (1e-2 * torch.randn(n, d, generator=g, device=DEV)).to(dt)
    return w, y, go


def _clip_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    b, t, d, v = case["batch"], case["seq"], case["width"], case["vocab"]
    y = _tokens(g, b * t, v).view(b, t)
    share = torch.rand(b, 1, generator=g, device=DEV) * 2 * case["padded"]
    pad = torch.arange(t, device=DEV).unsqueeze(0) >= t - (share * t).long()
    y[pad] = v - 1
    # Norms around the threshold: some examples are clipped, some are not.
    size = torch.exp(0.8 * torch.randn(b, 1, 1, generator=g, device=DEV)) / math.sqrt(t * d)
    go = (size * torch.randn(b, t, d, generator=g, device=DEV)).to(dt)
    return y, go


def prepare(case, seed):
    if case["kind"] == "loss":
        x, w, y = _loss_inputs(case, seed)
        return {"case": case, "x": x.requires_grad_(case["grad"] != "none"),
                "w": w.requires_grad_(case["grad"] == "xw"), "y": y}
    if case["kind"] == "lookup":
        w, y, go = _lookup_inputs(case, seed)
        return {"case": case, "w": w.requires_grad_(case["grad"]), "y": y, "go": go}
    y, go = _clip_inputs(case, seed)
    return {"case": case, "y": y, "go": go, "plan": None}


def _scale(case):
    return math.sqrt(case["width"]) if case["scaled"] else 1.0


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    return (_RUN_OWN if own else _RUN_PLAIN)[state["case"]["kind"]](state)


def _own_loss(s):
    from opaque_amd.vocabulary import linear_cross_entropy

    case = s["case"]
    loss = linear_cross_entropy(s["x"], s["w"], s["y"], softcap=case["softcap"] or None, ignore_index=IGNORE,
                                reduction="none" if case["grad"] == "none" else "mean")
    if case["grad"] == "none":
        return [loss]
    wanted = [s["x"], s["w"]] if case["grad"] == "xw" else [s["x"]]
    return [loss.detach(), *torch.autograd.grad(loss, wanted)]


def _plain_loss(s):
    case = s["case"]
    x, w, y = s["x"].detach().float(), s["w"].detach().float(), s["y"]
    live = y != IGNORE
    at = torch.where(live, y, 0).unsqueeze(1)
    z = x @ w.t()
    if case["softcap"]:
        z = case["softcap"] * torch.tanh(z / case["softcap"])
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    losses = torch.where(live, (torch.log(total) + top - z.gather(1, at)).squeeze(1), 0.0)
    if case["grad"] == "none":
        return [losses]
    count = live.sum()
    d = e / total
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=d.dtype))
    d = d * torch.where(live, 1.0 / count, 0.0).unsqueeze(1)
    if case["softcap"]:
        d = d * (1 - (z / case["softcap"]) ** 2)
    out = [losses.sum() / count, (d @ w).to(s["x"].dtype)]
    if case["grad"] == "xw":
        out.append((d.t() @ x).to(s["w"].dtype))
    return out


def _own_lookup(s):
    from opaque_amd.vocabulary import embedding

    out = embedding(s["y"], s["w"], scale=_scale(s["case"]))
    if not s["case"]["grad"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, [s["w"]], s["go"])]


def _plain_lookup(s):
    case, w = s["case"], s["w"].detach()
    out = (w[s["y"]].float() * _scale(case)).to(w.dtype)
    if not case["grad"]:
        return [out]
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, s["y"], s["go"].float())
    return [out, (dw * _scale(case)).to(w.dtype)]


def _own_clip(s):
    plan = s["plan"]
    if plan is None:  # the plan a training loop keeps from step to step
        from opaque_amd import _native as N
        from opaque_amd.engine import ClipSpec, EmbeddingSite, GhostPlan, LeafOut, Segments
        from opaque_amd.guard import guard_constants, leaf_guards

        case, dt = s["case"], s["go"].dtype
        shape = (case["vocab"], case["width"])
        _, rnd = leaf_guards([shape], [dt], None)
        clip = ClipSpec(mode=N.CLIP_AUTOS, thresholds=[1.0], effective=1.0, gamma=GAMMA,
                        normalize_by=float(case["batch"]), guards=[(*guard_constants(dt, rnd), dt)])
        plan = s["plan"] = GhostPlan(segments=Segments.padded(case["batch"], case["seq"]),
                                     leaves=[LeafOut(shape, dt)], clip=clip,
                                     embedding_sites=[EmbeddingSite(tokens=s["y"], g=s["go"], w_leaf=0)],
                                     device=s["go"].device)
    res = plan.run()
    return [res.leaves[0], res.norms]


def _held_factor(norms, dtype):
    """An example's AUTO-S factor as the table's type holds it, kept under the
    bound whichever way that type rounds: the definition's guard."""
    fi = torch.finfo(dtype)
    return (1.0 / (norms + GAMMA) * (1.0 - fi.eps - 2.0**-24) - fi.smallest_normal * fi.eps).to(dtype)


def _plain_clip(s):
    case, go = s["case"], s["go"]
    b, t, d, v = case["batch"], case["seq"], case["width"], case["vocab"]
    ex = torch.arange(b, device=go.device).repeat_interleave(t)
    pairs, where = torch.unique(ex * v + s["y"].reshape(-1), return_inverse=True)  # the (example, token) rows
    rows = torch.zeros(pairs.numel(), d, dtype=torch.float32, device=go.device)
    rows.index_add_(0, where, go.reshape(b * t, d).float())
    who = torch.div(pairs, v, rounding_mode="floor")
    sq = torch.zeros(b, dtype=torch.float32, device=go.device).index_add_(0, who, (rows * rows).sum(1))
    norms = torch.sqrt(sq)
    factor = _held_factor(norms, go.dtype).float()
    out = torch.zeros(v, d, dtype=torch.float32, device=go.device)
    out.index_add_(0, pairs - who * v, rows * factor[who].unsqueeze(1))
    return [(out / b).to(go.dtype), norms]


_RUN_OWN = {"loss": _own_loss, "lookup": _own_lookup, "clip": _own_clip}
_RUN_PLAIN = {"loss": _plain_loss, "lookup": _plain_lookup, "clip": _plain_clip}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_loss(case, seed):
    x, w, y = _loss_inputs(case, seed)
    x, w = x.double(), w.double()
    n = x.shape[0]
    live = (y != IGNORE).nonzero().squeeze(1)
    k = live.numel()
    losses = torch.zeros(n, dtype=torch.float64, device=DEV)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w) if case["grad"] == "xw" else None
    for rows in live.split(1024):
        u = x[rows] @ w.t()
        z = case["softcap"] * torch.tanh(u / case["softcap"]) if case["softcap"] else u
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        at = y[rows]
        losses[rows] = -logp.gather(1, at.unsqueeze(1)).squeeze(1)
        if case["grad"] == "none":
            continue
        p = logp.exp()
        p[torch.arange(rows.numel(), device=DEV), at] -= 1.0
        if case["softcap"]:
            p *= 1.0 - torch.tanh(u / case["softcap"]) ** 2
        p /= k
        dx[rows] = p @ w
        if dw is not None:
            dw += p.t() @ x[rows]
    if case["grad"] == "none":
        return [losses]
    out = [losses.sum() / k, dx]
    return out if dw is None else [*out, dw]


def _exact_lookup(case, seed):
    w, y, go = _lookup_inputs(case, seed)
    out = w.double()[y] * _scale(case)
    if not case["grad"]:
        return [out]
    order = torch.argsort(y, stable=True)
    toks, counts = torch.unique_consecutive(y[order], return_counts=True)
    total = torch.cumsum(go.double()[order], 0)
    ends = torch.cumsum(counts, 0) - 1
    upto = total[ends]
    sums = torch.cat([upto[:1], upto[1:] - upto[:-1]])
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    dw[toks] = sums * _scale(case)
    return [out, dw]


def _exact_clip(case, seed):
    y, go = _clip_inputs(case, seed)
    out = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device=DEV)
    norms = torch.zeros(case["batch"], dtype=torch.float64, device=DEV)
    dt = DTYPES[case["dtype"]]
    # The guard: the type's own rounding of the factor and the norm's (a
    # float32 square, a sum in 64 bits), and the type's least value.
    low, tiny = 1.0 - 2.0 * (torch.finfo(dt).eps / 2 + 2.0**-25), torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    for i in range(case["batch"]):
        toks, where = torch.unique(y[i], return_inverse=True)
        rows = torch.zeros(toks.numel(), case["width"], dtype=torch.float64, device=DEV)
        rows.index_add_(0, where, go[i].double())
        norms[i] = rows.square().sum().sqrt()
        out[toks] += rows * (low / (norms[i] + GAMMA) - tiny).to(dt).double()
    return [out / case["batch"], norms]


def exact(case, seed):
    return {"loss": _exact_loss, "lookup": _exact_lookup, "clip": _exact_clip}[case["kind"]](case, seed)
