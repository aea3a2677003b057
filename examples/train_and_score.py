"""A small language model's training step and next-token scores on the quantized
Linears and the operators between them (one MI355X).

    python examples/train_and_score.py [--steps N]

One channel-mix block over an embedding: layer norm over heads, layer norm, up
projection, squared ReLU, down projection, layer norm, output head, token log
probabilities with an entropy term.  Norms' and activation's inputs are kept in 8
bits for the backward pass, as the Linears keep theirs.  The data are synthetic: the
next token is a fixed function of the token.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pratchya_amd import functional as F            # noqa: E402
from pratchya_amd.qarr import QArrayImpl            # noqa: E402

BLK = 128
HEADS = 16


def init(vocab: int, hidden: int, inner: int, seed: int = 0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(torch.bfloat16).requires_grad_(True)

    def norm():
        return [torch.ones(hidden, device="cuda", requires_grad=True),
                torch.zeros(hidden, device="cuda", requires_grad=True)]
    return {"embed": normal(vocab, hidden, std=1.0), "heads": norm(), "mix": norm(), "last": norm(),
            "up": normal(hidden, inner, std=hidden ** -0.5), "down": normal(inner, hidden, std=inner ** -0.5),
            "head": normal(hidden, vocab, std=hidden ** -0.5)}


def linear(x: torch.Tensor, w: torch.Tensor, grid) -> torch.Tensor:
    return (QArrayImpl(x, (1, BLK)) @ QArrayImpl(w, grid)).astype(x.dtype)


def logits(p, tokens: torch.Tensor) -> torch.Tensor:
    """Logits of the next token, [n, vocab], for tokens [n]."""
    kept = (1, BLK)
    x = F.layer_norm(p["embed"][tokens], *p["heads"], groups=HEADS, tgrid=kept)
    h = F.layer_norm(x, *p["mix"], tgrid=kept)
    h = F.activation(linear(h, p["up"], (BLK, BLK)), "relu2", tgrid=kept)
    x = x + linear(h, p["down"], (BLK, BLK))
    return linear(F.layer_norm(x, *p["last"], tgrid=kept), p["head"], (BLK, 1))


def train_step(p, tokens: torch.Tensor, targets: torch.Tensor, lr: float = 0.5) -> torch.Tensor:
    """One step of gradient descent; targets below 0 are left out.  Returns the mean loss."""
    out = F.token_logprobs(logits(p, tokens), targets, entropy=True)
    n = (targets >= 0).sum().clamp(min=1)
    loss = -out.logprobs.sum() / n
    leaves = [t for v in p.values() for t in (v if isinstance(v, list) else [v])]
    grads = torch.autograd.grad(loss - 0.001 * out.entropy.mean(), leaves)
    with torch.no_grad():
        for t, g in zip(leaves, grads):
            t.sub_((lr * g / (g.float().norm() + 1e-6) * t.float().norm() * 0.02).to(t.dtype))
    return loss.detach()


def score(p, tokens: torch.Tensor, targets: torch.Tensor, top: int = 5) -> F.TokenLogprobs:
    """Log probabilities of targets, entropies and the best alternatives, without gradients."""
    with torch.no_grad():
        return F.token_logprobs(logits(p, tokens), targets, entropy=True, top=top)


def batch(vocab: int, n: int, step: int):
    gen = torch.Generator(device="cuda").manual_seed(1000 + step)
    tokens = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    targets = (tokens * 7 + 3) % vocab
    # the first positions belong to a prompt
    return tokens, torch.where(torch.arange(n, device="cuda") < n // 16, -1, targets)


def main(steps: int = 30, vocab: int = 512, hidden: int = 1024, inner: int = 2048, rows: int = 1024):
    p = init(vocab, hidden, inner)
    losses = [train_step(p, *batch(vocab, rows, i)) for i in range(steps)]
    tokens, targets = batch(vocab, 8, -1)
    return p, torch.stack(losses), score(p, tokens, targets)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    _, losses, scores = main(ap.parse_args().steps)
    for i, v in enumerate(losses.tolist()):
        if i % 5 == 0 or i == len(losses) - 1:
            print(f"step {i:3d}  loss {v:.4f}")
    for row in range(len(scores.logprobs)):
        best = ", ".join(f"{t}: {v:.3f}" for t, v in zip(scores.top_tokens[row].tolist(), scores.top_logprobs[row].tolist()))
        print(f"log probability {scores.logprobs[row]:.4f}  entropy {scores.entropy[row]:.4f}  best {best}")
