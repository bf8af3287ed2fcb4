"""DP-SGD training of a small language model whose every weight trains, vocabulary ends included.

The model is an embedding, gated blocks of full-weight linears and an output
head.  Inside ``clipped_grad`` its tables and weights are seams: the
embedding's per-example norms and clipped sum come from tokens and output
gradients (``EmbeddingSite``), the linears' and the head's from activations
and output gradients, and the loss never holds [tokens, vocabulary] logits in
float32.  No [examples, vocabulary, width] gradient exists.

    python examples/dp_language_model.py [--vocab 32000 --width 1024 --steps 20]

Data is synthetic: sequences in which a token follows another by a fixed
permutation, after a prompt that bears no loss, padded at the end.
"""

from __future__ import annotations

import argparse
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import torch

from opaque_amd.capture import linear
from opaque_amd.clipping import auto_clipped_grad
from opaque_amd.noise import gaussian_noise
from opaque_amd.random import key
from opaque_amd.vocabulary import embedding, linear_cross_entropy

PAD = 0
IGNORE = -100


def init(vocab: int, width: int, blocks: int, seed: int, device="cuda", dtype=torch.bfloat16) -> dict:
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(rows, cols, std):
        return (std * torch.randn(rows, cols, generator=g, device=device)).to(dtype)

    params = {"embed": normal(vocab, width, width**-0.5), "head": normal(vocab, width, width**-0.5)}
    for b in range(blocks):
        params[f"in{b}"] = normal(4 * width, width, width**-0.5)
        params[f"out{b}"] = normal(width, 2 * width, (2 * width) ** -0.5)
    return params


def loss_fn(params: dict, tokens: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """The mean loss of one example's tokens."""
    width = params["embed"].shape[1]
    h = embedding(tokens, params["embed"], scale=width**0.5, padding_idx=PAD)
    for b in range(sum(k.startswith("in") for k in params)):
        gate, up = linear(h, params[f"in{b}"]).chunk(2, -1)
        h = h + linear(torch.nn.functional.silu(gate) * up, params[f"out{b}"])
    h = torch.nn.functional.rms_norm(h.float(), (width,)).to(h.dtype)
    return linear_cross_entropy(h, params["head"], target, softcap=30.0, ignore_index=IGNORE)


def batch(n: int, seq: int, follow: torch.Tensor, seed: int):
    """Tokens and targets [n, seq]: each token's successor, none for the prompt and the padding."""
    g = torch.Generator().manual_seed(seed)
    vocab = follow.numel()
    tokens = torch.empty(n, seq + 1, dtype=torch.int64)
    tokens[:, 0] = torch.randint(1, vocab, (n,), generator=g)
    for t in range(seq):
        tokens[:, t + 1] = follow[tokens[:, t]]
    target = tokens[:, 1:].clone()
    tokens = tokens[:, :-1].clone()
    length = torch.randint(seq // 2 + 1, seq + 1, (n, 1), generator=g)
    place = torch.arange(seq).unsqueeze(0)
    tokens[place >= length] = PAD
    target[(place >= length) | (place < seq // 8)] = IGNORE
    return tokens.cuda(), target.cuda()


def train(vocab=2048, width=256, blocks=2, examples=16, seq=64, steps=20, lr=0.05, noise=0.1, report=print) -> list:
    """The losses of ``steps`` DP steps."""
    follow = torch.cat([torch.zeros(1, dtype=torch.int64),
                        1 + torch.randperm(vocab - 1, generator=torch.Generator().manual_seed(7))])
    params = init(vocab, width, blocks, seed=0)
    grad_fn, clip_state = auto_clipped_grad(loss_fn, R=1.0, normalize_by=float(examples), batch_argnums=(1, 2),
                                            return_aux=True)
    noise_fn, noise_state = gaussian_noise(noise_multiplier=noise, key=key(1))
    losses = []
    for step in range(steps):
        tokens, target = batch(examples, seq, follow, seed=step % 4)
        began = time.perf_counter()
        (grads, aux), clip_state = grad_fn(params, tokens, target, state=clip_state)
        noisy, noise_state = noise_fn(grads, noise_state)
        params = {k: (p.float() - lr * width**0.5 * noisy.pytree[k].float()).to(p.dtype) for k, p in params.items()}
        losses.append(float(aux.loss_values.mean()))
        report(f"step {step}: loss {losses[-1]:.4f}, median norm {float(aux.grad_norms.median()):.3f}, "
               f"{(time.perf_counter() - began) * 1e3:.1f} ms")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("vocab", 2048), ("width", 256), ("blocks", 2), ("examples", 16), ("seq", 64), ("steps", 20)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--lr", type=float, default=0.05)
    ap.add_argument("--noise", type=float, default=0.1)
    train(**vars(ap.parse_args()))
