"""A small linear-attention language model on the quantized Linears and the operators
around them: a training step over a padded batch, and generation (one MI355X).

    python examples/linear_attention_lm.py [--steps N]

The embedding table serves as the output head.  One block of time mixing: layer norm, one
projection to queries, keys, values and the tokens' decays, linear attention, layer norm
over heads, output projection.  The loss is the head's cross entropy, whose logits are not
kept.  Generation reads a prompt with ``linear_attention`` and goes on token by token from
the state that it returns, updated in place.  The data are synthetic: a token follows the
one some places before it.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pratchya_amd import functional as F            # noqa: E402
from pratchya_amd.qarr import QArrayImpl            # noqa: E402

BLK = 128
HEAD = 64


def init(vocab: int, hidden: int, seed: int = 0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(torch.bfloat16).requires_grad_(True)

    def norm():
        return [torch.ones(hidden, device="cuda", requires_grad=True),
                torch.zeros(hidden, device="cuda", requires_grad=True)]
    heads = hidden // HEAD
    # heads forget half after one token to hundreds
    slow = torch.linspace(0.0, 6.0, heads, device="cuda").requires_grad_(True)
    return {"embed": normal(vocab, hidden, std=hidden ** -0.5), "mix": norm(), "heads": norm(), "last": norm(),
            "qkv": normal(hidden, 3 * hidden, std=hidden ** -0.5), "out": normal(hidden, hidden, std=hidden ** -0.5),
            "gate": normal(hidden, BLK * -(-heads // BLK), std=hidden ** -0.5), "slow": slow}


def linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return (QArrayImpl(x, (1, BLK)) @ QArrayImpl(w, (BLK, BLK))).astype(x.dtype)


def mix_inputs(p, x: torch.Tensor):
    """Queries, keys, values [..., heads, HEAD] and log decays [..., heads] of rows x [..., hidden]."""
    rows = x.reshape(-1, x.shape[-1])
    h = F.layer_norm(rows, *p["mix"])
    heads = x.shape[-1] // HEAD
    q, k, v = linear(h, p["qkv"]).unflatten(0, x.shape[:-1]).unflatten(-1, (3 * heads, HEAD)).split(heads, dim=-2)
    gate = linear(h, p["gate"])[:, :heads].unflatten(0, x.shape[:-1])
    return q, k, v, -torch.exp(-p["slow"]) * torch.sigmoid(gate.float())


def mix_output(p, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
    rows = o.reshape(-1, x.shape[-1])
    y = linear(F.layer_norm(rows, *p["heads"], groups=x.shape[-1] // HEAD), p["out"]).reshape(x.shape)
    return F.layer_norm((x + y).reshape(-1, x.shape[-1]), *p["last"]).reshape(x.shape)


def hidden_rows(p, tokens: torch.Tensor, lengths=None, state=None):
    """Rows that the head reads [B, T, hidden], and the state behind each sequence."""
    x = F.embedding(p["embed"], tokens, scale=math.sqrt(p["embed"].shape[1]))
    r = F.linear_attention(*mix_inputs(p, x), state=state, lengths=lengths, scale=HEAD ** -0.5)
    return mix_output(p, x, r.out), r.state


def losses(p, tokens: torch.Tensor, targets: torch.Tensor, lengths=None) -> torch.Tensor:
    """Cross entropy of each target (0 for those below 0), [B, T]."""
    h, _ = hidden_rows(p, tokens, lengths)
    return F.linear_cross_entropy(h, p["embed"].t(), targets, label_smoothing=0.05)


def leaves(p):
    return [t for v in p.values() for t in (v if isinstance(v, list) else [v])]


def train_step(p, tokens, targets, lengths, lr: float = 0.5) -> torch.Tensor:
    """One step of gradient descent.  Returns the mean loss."""
    loss = losses(p, tokens, targets, lengths).sum() / (targets >= 0).sum().clamp(min=1)
    grads = torch.autograd.grad(loss, leaves(p))
    with torch.no_grad():
        for t, g in zip(leaves(p), grads):
            t.sub_((lr * g / (g.float().norm() + 1e-6) * t.float().norm() * 0.02).to(t.dtype))
    return loss.detach()


def step_rows(p, tokens: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """The head's rows [B, hidden] of one more token of each sequence; state is updated in place."""
    x = F.embedding(p["embed"], tokens, scale=math.sqrt(p["embed"].shape[1]))
    return mix_output(p, x, F.linear_attention_step(*mix_inputs(p, x), state, scale=HEAD ** -0.5))


@torch.no_grad()
def generate(p, prompt: torch.Tensor, lengths: torch.Tensor, count: int):
    """The most probable `count` tokens behind prompts [B, T] of some lengths, [B, count]."""
    h, state = hidden_rows(p, prompt, lengths)
    row = h[torch.arange(len(prompt), device=h.device), lengths - 1]
    found = []
    for _ in range(count):
        found.append((row @ p["embed"].t()).float().argmax(dim=-1))
        row = step_rows(p, found[-1], state)
    return torch.stack(found, dim=1)


def batch(vocab: int, batch: int, length: int, step: int, back: int = 3):
    """Tokens that repeat with a period, their successors, and the sequences' lengths; what lies behind has no target."""
    gen = torch.Generator(device="cuda").manual_seed(1000 + step)
    period = torch.randint(0, vocab, (batch, back), generator=gen, device="cuda")
    t = period.repeat(1, length // back + 2)
    lengths = torch.randint(length // 2, length + 1, (batch,), generator=gen, device="cuda")
    here = torch.arange(length, device="cuda") < lengths[:, None]
    return t[:, :length].contiguous(), torch.where(here, t[:, 1:length + 1], -1), lengths


def main(steps: int = 30, vocab: int = 512, hidden: int = 1024, rows: int = 8, length: int = 200):
    p = init(vocab, hidden)
    out = [train_step(p, *batch(vocab, rows, length, i)) for i in range(steps)]
    tokens, _, lengths = batch(vocab, 4, 64, -1)
    return p, torch.stack(out), generate(p, tokens, lengths, 6)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    _, found, tokens = main(ap.parse_args().steps)
    for i, v in enumerate(found.tolist()):
        if i % 5 == 0 or i == len(found) - 1:
            print(f"step {i:3d}  loss {v:.4f}")
    print("generated", tokens.tolist())
