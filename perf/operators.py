"""The operators around the quantized Linears, as cases that can be timed and checked.

Layer norm with its gradients, activations whose input is kept in 8 bits for
the backward pass, and log probabilities of tokens with entropy, top
alternatives and the logits' gradient.  ``run`` computes them with elementary
torch operations in 32 bits, or, where ``own`` is true, through
``pratchya_amd.functional`` as a model's code calls it.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # one token of generation through a 4096-wide model's norm
        {"name": "norm token", "op": "norm", "rows": 1, "width": 4096, "groups": 1, "dtype": "bf16", "train": False,
         "blk": 0},
        # the norm over each head of 64 after the time mixing, training step of a batch
        {"name": "norm heads", "op": "norm", "rows": 8192, "width": 4096, "groups": 64, "dtype": "bf16",
         "train": True, "blk": 0},
        # rows that no vector width divides, in 32 bits
        {"name": "norm odd", "op": "norm", "rows": 1001, "width": 2057, "groups": 1, "dtype": "f32", "train": True,
         "blk": 0},
        # a batch's residual stream in a 4096-wide model, kept in 8 bits for the backward pass
        {"name": "norm", "op": "norm", "rows": 16384, "width": 4096, "groups": 1, "dtype": "bf16", "train": True,
         "blk": 128},
        # a short sequence's activation, blocks of the 32-wide preset
        {"name": "activation short", "op": "act", "kind": "silu", "rows": 128, "width": 8192, "dtype": "bf16",
         "blk": 32},
        # a ragged prompt whose width is an odd number of blocks: scale groups run over the rows' ends
        {"name": "activation ragged", "op": "act", "kind": "gelu", "rows": 1000, "width": 2176, "dtype": "f32",
         "blk": 128},
        # the up-projection's output of a 2048-wide model, without 8-bit storage
        {"name": "activation kept", "op": "act", "kind": "relu2", "rows": 4096, "width": 8192, "dtype": "bf16",
         "blk": 0},
        # the up-projection's output of a batch in a 4096-wide model
        {"name": "activation", "op": "act", "kind": "relu2", "rows": 16384, "width": 16384, "dtype": "bf16",
         "blk": 128},
        # one generated token: its log probability, the entropy and the 20 best alternatives
        {"name": "score token", "op": "logp", "rows": 1, "vocab": 65536, "dtype": "bf16", "train": False,
         "entropy": True, "top": 20, "pad": 0},
        # a batch of sequences' next tokens with 5 alternatives, 32-bit logits of a padded vocabulary
        {"name": "score batch", "op": "logp", "rows": 256, "vocab": 32768, "dtype": "f32", "train": False,
         "entropy": False, "top": 5, "pad": 100},
        # the loss of a ragged batch over a vocabulary of odd size
        {"name": "loss odd", "op": "logp", "rows": 1000, "vocab": 50021, "dtype": "f32", "train": True,
         "entropy": False, "top": 0, "pad": 0},
        # a training step's loss with an entropy term over the 65536-token head
        {"name": "loss", "op": "logp", "rows": 8192, "vocab": 65536, "dtype": "bf16", "train": True, "entropy": True,
         "top": 0, "pad": 0},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "act", "logp", "logp"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        form = rng.choice(["plain", "heads", "stored"])
        case = {"op": "norm", "rows": _between(rng, 1, 16384), "width": _between(rng, 32, 8192), "groups": 1,
                "dtype": dtype, "train": rng.random() < 0.75, "blk": 0}
        if form == "heads":
            head = rng.choice([32, 64, 128, _between(rng, 16, 256)])
            case["groups"] = _between(rng, 1, 64)
            case["width"] = head * case["groups"]
        elif form == "stored":
            case["blk"] = rng.choice([128, 128, 32, 16])
            case["width"] = case["blk"] * max(1, case["width"] // case["blk"])
            case["train"] = True
        return case
    if op == "act":
        blk = rng.choice([128, 128, 32, 16, 0])
        width = _between(rng, 128, 16384)
        return {"op": "act", "kind": rng.choice(["relu2", "silu", "gelu"]), "rows": _between(rng, 1, 8192),
                "width": blk * max(1, width // blk) if blk else width, "dtype": dtype, "blk": blk}
    if rng.random() < 0.5:
        vocab = _between(rng, 100, 65536)
        return {"op": "logp", "rows": _between(rng, 1, 4096), "vocab": vocab, "dtype": dtype, "train": True,
                "entropy": rng.random() < 0.5, "top": 0, "pad": rng.choice([0, 0, vocab // 64])}
    vocab = _between(rng, 100, 131072)
    return {"op": "logp", "rows": _between(rng, 1, 512), "vocab": vocab, "dtype": dtype, "train": False,
            "entropy": rng.random() < 0.5, "top": rng.choice([1, 5, 20, 64]), "pad": rng.choice([0, 0, vocab // 64])}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    rows = case["rows"]
    if case["op"] == "logp":
        vocab, pad = case["vocab"], case["pad"]
        x = torch.randn((rows, vocab), generator=gen, device=DEV, dtype=dtype).mul_(2.5)
        tokens = torch.randint(0, vocab - pad, (rows,), generator=gen, device=DEV)
        # the model has learnt something: the token that came stands out
        x.scatter_(1, tokens[:, None], (_normal(gen, rows, 1) + 8).to(dtype))
        if pad:
            x[:, vocab - pad:] = -math.inf
        if case["train"]:
            # positions of a prompt carry no token
            tokens = torch.where(torch.rand((rows,), generator=gen, device=DEV) < 0.02, -1, tokens)
            s["g"] = _normal(gen, rows) / rows
            s["gh"] = torch.full((rows,), 0.01 / rows, device=DEV)
            x.requires_grad_(True)
        s["x"], s["tokens"] = x, tokens
        return s
    width = case["width"]
    # 1% of the channels 20 times larger, as transformer activations have them
    big = torch.where(torch.rand((1, width), generator=gen, device=DEV) < 0.01, 20.0, 1.0)
    s["x"] = (_normal(gen, rows, width) * big + 0.1).to(dtype)
    if case["op"] == "norm":
        s["w"] = 1 + 0.1 * _normal(gen, width)
        s["b"] = 0.1 * _normal(gen, width)
    if case["op"] == "act" or case["train"]:
        s["g"] = (_normal(gen, rows, width) * 1e-3).to(dtype)
        for n in ("x", "w", "b"):
            if n in s:
                s[n].requires_grad_(True)
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return (_run_own if own else {"norm": _norm, "act": _act, "logp": _logp}[case["op"]])(state, case)


def _run_own(s, case):
    from pratchya_amd import functional as F
    tgrid = (1, case["blk"]) if case.get("blk") else None
    if case["op"] == "norm":
        y = F.layer_norm(s["x"], s["w"], s["b"], eps=EPS, groups=case["groups"], tgrid=tgrid)
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"])
    if case["op"] == "act":
        y = F.activation(s["x"], case["kind"], tgrid=tgrid)
        return (y.detach(),) + torch.autograd.grad(y, (s["x"],), s["g"])
    r = F.token_logprobs(s["x"], s["tokens"], entropy=case["entropy"], top=case["top"])
    out = {"logprobs": r.logprobs.detach()}
    if case["entropy"]:
        out["entropy"] = r.entropy.detach()
    if case["top"]:
        out["top"], out["top tokens"] = r.top_logprobs, r.top_tokens
    if case["train"]:
        ends = (r.logprobs, r.entropy) if case["entropy"] else (r.logprobs,)
        out["dx"], = torch.autograd.grad(ends, (s["x"],), (s["g"], s["gh"])[:len(ends)])
    return out


def _stored(x, blk):
    """A 32-bit [rows, width] x as its 8-bit form with block grid (1, blk) stands for it."""
    if not blk:
        return x
    m = x.reshape(-1, blk).abs().amax(dim=1)
    k = math.gcd(max(1, blk // 16), m.numel())
    top = m.reshape(-1, k).amax(dim=1, keepdim=True)
    ratio = m.reshape(-1, k) / torch.where(top == 0, 1.0, top)
    power = (ratio.view(torch.int32) & 0x7F800000).view(torch.float32)
    scale = (power * top).reshape(-1, 1)
    q = (x.reshape(-1, blk) / scale.clamp(min=1e-7) * 128).to(torch.bfloat16).to(torch.float8_e4m3fn)
    return (q.float() * scale / 128).reshape(x.shape)


def _norm(s, case):
    dtype, groups = s["x"].dtype, case["groups"]
    w, b = s["w"].detach().float(), s["b"].detach().float()
    x = s["x"].detach().float()
    rows, width = x.shape
    seg = x.reshape(rows, groups, -1)
    mean = seg.mean(dim=2, keepdim=True)
    rstd = ((seg - mean) ** 2).mean(dim=2, keepdim=True).add(EPS).rsqrt()
    y = ((seg - mean) * rstd).reshape(rows, width) * w + b
    if not case["train"]:
        return y.to(dtype)
    h = (_stored(x, case["blk"]).reshape(seg.shape) - mean) * rstd
    g = s["g"].float()
    a = (g * w).reshape(seg.shape)
    dx = rstd * (a - a.mean(dim=2, keepdim=True) - h * (a * h).mean(dim=2, keepdim=True))
    dw = (g * h.reshape(rows, width)).sum(dim=0)
    return y.to(dtype), dx.reshape(rows, width).to(dtype), dw.to(s["w"].dtype), g.sum(dim=0).to(s["b"].dtype)


def _act(s, case):
    dtype, kind = s["x"].dtype, case["kind"]
    x = s["x"].detach().float()
    v = _stored(x, case["blk"])
    if kind == "relu2":
        y, d = x.clamp(min=0) ** 2, 2 * v.clamp(min=0)
    elif kind == "silu":
        p = 1 / (1 + torch.exp(-v))
        y, d = x / (1 + torch.exp(-x)), p * (1 + v * (1 - p))
    else:
        y = x * 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        d = 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    return y.to(dtype), (d * s["g"].float()).to(dtype)


def _logp(s, case):
    tokens, top = s["tokens"], case["top"]
    x = s["x"].detach().float()
    vocab = x.shape[1]
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    d = x - m
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    logs = torch.log(total)
    here, at = tokens >= 0, tokens.clamp(min=0)[:, None]
    logp = (d.gather(1, at) - logs).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)[:, 0]
    out = {"logprobs": torch.where(here, logp, 0.0)}
    safe = torch.where(total == 0, 1.0, total)
    if case["entropy"]:
        h = torch.log(safe) - torch.where(e > 0, e * d, 0.0).sum(dim=1, keepdim=True) / safe
        out["entropy"] = h[:, 0]
    if top:
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (order << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
        best = torch.topk(key, top, dim=1, sorted=True).values
        found = vocab - 1 - (best & 0xFFFFFFFF)
        out["top"], out["top tokens"] = d.gather(1, found) - logs, found
    if case["train"]:
        g = torch.where(here, s["g"], 0.0)[:, None]
        p = e / safe
        dx = -p * g
        if case["entropy"]:
            dx = dx - torch.where(e > 0, p * (d - torch.log(safe) + h), 0.0) * s["gh"][:, None]
        dx.scatter_add_(1, at, g)
        out["dx"] = dx.to(s["x"].dtype)
    return out


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    rows = case["rows"]
    if case["op"] == "logp":
        n = rows * case["vocab"]
        small = rows * (8 + 4 + 4 * case["entropy"] + 12 * case["top"] + 8 * case["train"])
        return {"bytes": e * n * (2 if case["train"] else 1) + small, "flops": n * (10 if case["train"] else 4)}
    n = rows * case["width"]
    if case["op"] == "act":
        return {"bytes": 4 * e * n, "flops": 8 * n}
    params = 4 * case["width"]
    return {"bytes": (4 * e * n + 4 * params) if case["train"] else (2 * e * n + 2 * params),
            "flops": (20 if case["train"] else 8) * n}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _exact_stored(x, blk):
    """What the 8-bit form of x holds, in 64 bits: a block's scale is a power of two of its group's largest
    value; quotients are 32-bit values rounded to bf16 and from there to e4m3."""
    if not blk:
        return x.double()
    blocks = x.float().reshape(-1, blk)
    m = blocks.abs().max(dim=1).values
    k = math.gcd(max(1, blk // 16), len(m))
    group = m.reshape(-1, k).max(dim=1).values.repeat_interleave(k)
    ratio = m / torch.where(group > 0, group, 1)
    scale = torch.ldexp(torch.ones_like(ratio).double(), torch.frexp(ratio).exponent - 1) * group.double()
    scale = torch.where(ratio >= 2.0 ** -126, scale, 0)[:, None]
    q = (blocks / scale.float().clamp(min=1e-7) * 128).to(torch.bfloat16).to(torch.float8_e4m3fn)
    return (q.double() * scale / 128).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    if case["op"] == "norm":
        seg = x.double().reshape(len(x), case["groups"], -1)
        var, mean = torch.var_mean(seg, dim=2, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        w, b = s["w"].detach().double(), s["b"].detach().double()
        y = ((seg - mean) / sd).reshape(x.shape) * w + b
        if not case["train"]:
            return y
        h = (_exact_stored(x, case["blk"]).reshape(seg.shape) - mean) / sd
        g = s["g"].double()
        a = (g * w).reshape(seg.shape)
        n = seg.shape[2]
        dx = (a - a.sum(2, keepdim=True) / n - h * (a * h).sum(2, keepdim=True) / n) / sd
        return y, dx.reshape(x.shape), torch.einsum("rc,rc->c", g, h.reshape(x.shape)), g.sum(0)
    if case["op"] == "act":
        v, u, g = _exact_stored(x, case["blk"]), x.double(), s["g"].double()
        if case["kind"] == "relu2":
            return torch.where(u > 0, u * u, 0), torch.where(v > 0, 2 * v, 0) * g
        if case["kind"] == "silu":
            p = torch.sigmoid(v)
            return u * torch.sigmoid(u), p * (1 + v * torch.sigmoid(-v)) * g
        phi = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        return u * torch.special.ndtr(u), (torch.special.ndtr(v) + v * phi) * g
    u, tokens = x.double(), s["tokens"]
    lse = torch.logsumexp(u, dim=1, keepdim=True)
    here, at = tokens >= 0, tokens.clamp(min=0)[:, None]
    out = {"logprobs": torch.where(here, (u.gather(1, at) - lse)[:, 0], 0)}
    p = torch.exp(u - lse)
    finite = torch.where(p > 0, u - lse, 0)
    h = -(p * finite).sum(1, keepdim=True)
    if case["entropy"]:
        out["entropy"] = h[:, 0]
    if case["top"]:
        order = torch.sort(u, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top"], out["top tokens"] = u.gather(1, order) - lse, order
    if case["train"]:
        g = torch.where(here, s["g"], 0).double()[:, None]
        dx = -g * p
        if case["entropy"]:
            dx = dx - s["gh"].double()[:, None] * p * (finite + h)
        out["dx"] = dx.scatter_add(1, at, g)
    return out
