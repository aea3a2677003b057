"""The operators at a model's two ends and in its time mixing, as cases that can be timed and checked.

Embedding lookup with scaling and the table's gradient, linear attention with a
decay for each head and token (chunks for prompts and training, one token at a
time for generation), and the cross entropy of an output head whose logits are
not kept, each with its gradients.  ``run`` computes them with elementary torch
operations in 32 bits, or, where ``own`` is true, through
``pratchya_amd.functional`` as a model's code calls it.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the tokens of one generation step of a batch
        {"name": "embed step", "op": "embed", "n": 64, "vocab": 65536, "width": 4096, "dtype": "bf16", "train": False},
        # a ragged batch over a vocabulary and a width that no vector divides, in 32 bits
        {"name": "embed odd", "op": "embed", "n": 1001, "vocab": 50021, "width": 2057, "dtype": "f32", "train": True},
        # a training batch's tokens: common ones come thousands of times
        {"name": "embed", "op": "embed", "n": 16384, "vocab": 65536, "width": 2048, "dtype": "bf16", "train": True},
        # one sequence's next token
        {"name": "mix token", "op": "step", "batch": 1, "heads": 32, "dk": 64, "dv": 64, "dtype": "bf16"},
        # a batch of sequences' next tokens
        {"name": "mix tokens", "op": "step", "batch": 128, "heads": 64, "dk": 64, "dv": 64, "dtype": "bf16"},
        # one long prompt that goes on from a state
        {"name": "mix prompt", "op": "mix", "batch": 1, "length": 8192, "heads": 64, "dk": 64, "dv": 64,
         "dtype": "bf16", "train": False, "carry": True, "ragged": False},
        # a padded batch of sequences of odd lengths in 32 bits, gradients through the states
        {"name": "mix odd", "op": "mix", "batch": 5, "length": 1001, "heads": 12, "dk": 48, "dv": 80, "dtype": "f32",
         "train": True, "carry": True, "ragged": True},
        # a training step's time mixing in a 2048-wide model
        {"name": "mix", "op": "mix", "batch": 8, "length": 4096, "heads": 32, "dk": 64, "dv": 64, "dtype": "bf16",
         "train": True, "carry": False, "ragged": False},
        # the loss of a short text, without gradients
        {"name": "head score", "op": "loss", "n": 128, "vocab": 32768, "width": 2048, "dtype": "bf16", "train": False,
         "smooth": 0.0, "tied": False},
        # a ragged batch over a vocabulary and a width of odd size in 32 bits
        {"name": "head odd", "op": "loss", "n": 1000, "vocab": 50021, "width": 1027, "dtype": "f32", "train": True,
         "smooth": 0.0, "tied": False},
        # a training step whose head is the embedding table, with smoothed labels
        {"name": "head tied", "op": "loss", "n": 4096, "vocab": 65536, "width": 2048, "dtype": "bf16", "train": True,
         "smooth": 0.1, "tied": True},
        # a training step's loss over the 65536-token head of a 4096-wide model
        {"name": "head", "op": "loss", "n": 8192, "vocab": 65536, "width": 4096, "dtype": "bf16", "train": True,
         "smooth": 0.0, "tied": False},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "step", "mix", "mix", "loss", "loss"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "embed":
        return {"op": "embed", "n": _between(rng, 1, 32768), "vocab": _between(rng, 100, 131072),
                "width": _between(rng, 32, 4096), "dtype": dtype, "train": rng.random() < 0.7}
    if op == "loss":
        width, vocab = _between(rng, 64, 4096), _between(rng, 100, 65536)
        if rng.random() < 0.7:      # as most models have them
            width, vocab = max(64, width // 64 * 64), max(128, vocab // 128 * 128)
        return {"op": "loss", "n": _between(rng, 1, 8192), "vocab": vocab, "width": width, "dtype": dtype,
                "train": rng.random() < 0.75, "smooth": rng.choice([0.0, 0.0, 0.1]), "tied": rng.random() < 0.5}
    form = rng.choice(["64", "64", "128", "any"])
    dk, dv = {"64": (64, 64), "128": (128, 128)}.get(form) or (rng.randint(16, 128), rng.randint(16, 128))
    heads = rng.choice([1, 12, 16, 32, 64])
    if op == "step":
        return {"op": "step", "batch": _between(rng, 1, 256), "heads": heads, "dk": dk, "dv": dv, "dtype": dtype}
    batch, length = _between(rng, 1, 16), _between(rng, 1, 8192)
    while batch * length * heads > 1 << 20:
        length = max(1, length // 2)
    return {"op": "mix", "batch": batch, "length": length, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype,
            "train": rng.random() < 0.6, "carry": rng.random() < 0.5, "ragged": rng.random() < 0.3}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _tokens(gen, n, vocab):
    """Tokens as text has them: the k-th most common one about 1 / k as often as the first."""
    u = torch.rand((n,), generator=gen, device=DEV, dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab + 1.0)).long().clamp(1, vocab) - 1
    return (rank * 40503 + 7) % vocab


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "embed":
        s["table"] = torch.randn((case["vocab"], case["width"]), generator=gen, device=DEV, dtype=dtype)
        s["tokens"] = _tokens(gen, case["n"], case["vocab"])
        s["scale"] = math.sqrt(case["width"])
        if case["train"]:
            s["table"].requires_grad_(True)
            s["g"] = (_normal(gen, case["n"], case["width"]) * 1e-3).to(dtype)
        return s
    if case["op"] == "loss":
        n, vocab, width = case["n"], case["vocab"], case["width"]
        s["x"] = _normal(gen, n, width).to(dtype)
        # the table's rows are the vocabulary's, the head's weight is [width, vocab]
        w = torch.randn((vocab, width) if case["tied"] else (width, vocab), generator=gen, device=DEV, dtype=dtype)
        w.mul_(2.0 / math.sqrt(width))
        s["w"], s["targets"] = w, _tokens(gen, n, vocab)
        if case["train"]:
            # positions of a prompt carry no target
            s["targets"] = torch.where(torch.rand((n,), generator=gen, device=DEV) < 0.02, -1, s["targets"])
            s["g"] = torch.full((n,), 1.0 / n, device=DEV)
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
        return s
    batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    lead = (batch, heads) if case["op"] == "step" else (batch, case["length"], heads)
    for name, d in (("q", dk), ("k", dk), ("v", dv)):
        s[name] = _normal(gen, *lead, d).to(dtype)
    # heads remember from a few tokens to about a thousand
    slow = torch.exp(-torch.linspace(0.7, 6.9, heads, device=DEV))
    s["decay"] = -slow * (0.5 + torch.rand(lead, generator=gen, device=DEV))
    s["scale"] = dk ** -0.5
    if case["op"] == "step" or case["carry"]:
        s["state"] = _normal(gen, batch, heads, dk, dv)
    if case["op"] == "step":
        return s
    if case["ragged"]:
        s["lengths"] = torch.randint(0, case["length"] + 1, (batch,), generator=gen, device=DEV)
        s["lengths"][:1] = case["length"]
    if case["train"]:
        s["g"] = _normal(gen, *lead, dv).to(dtype)
        if case["carry"]:
            s["gs"] = _normal(gen, batch, heads, dk, dv)
        for name in _leaves(s):
            s[name].requires_grad_(True)
    return s


def _leaves(s):
    return [n for n in ("q", "k", "v", "decay", "state") if n in s]


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return (_run_own if own else {"embed": _embed, "step": _step, "mix": _mix, "loss": _loss}[case["op"]])(state, case)


def _run_own(s, case):
    from pratchya_amd import functional as F
    if case["op"] == "embed":
        y = F.embedding(s["table"], s["tokens"], scale=s["scale"])
        return (y.detach(),) + (torch.autograd.grad(y, (s["table"],), s["g"]) if case["train"] else ())
    if case["op"] == "step":
        y = F.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], scale=s["scale"])
        return {"out": y, "state": s["state"]}
    if case["op"] == "mix":
        r = F.linear_attention(s["q"], s["k"], s["v"], s["decay"], state=s.get("state"), lengths=s.get("lengths"),
                               scale=s["scale"])
        out = {"out": r.out.detach(), "state": r.state.detach()}
        if case["train"]:
            leaves = _leaves(s)
            ends, gs = ((r.out, r.state), (s["g"], s["gs"])) if case["carry"] else ((r.out,), (s["g"],))
            out.update(zip(leaves_named(leaves), torch.autograd.grad(ends, [s[n] for n in leaves], gs)))
        return out
    w = s["w"].t() if case["tied"] else s["w"]
    y = F.linear_cross_entropy(s["x"], w, s["targets"], label_smoothing=case["smooth"])
    return (y.detach(),) + (torch.autograd.grad(y, (s["x"], s["w"]), s["g"]) if case["train"] else ())


def leaves_named(leaves):
    return ["d" + n for n in leaves]


def _embed(s, case):
    table, tokens = s["table"].detach(), s["tokens"]
    y = (table[tokens].float() * s["scale"]).to(table.dtype)
    if not case["train"]:
        return (y,)
    d = torch.zeros(table.shape, device=DEV)
    d.index_add_(0, tokens, s["g"].float() * s["scale"])
    return y, d.to(table.dtype)


def _step(s, case):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    s["state"].mul_(torch.exp(s["decay"])[..., None, None]).add_(k[..., :, None] * v[..., None, :])
    y = (q[..., :, None] * s["state"]).sum(dim=-2) * s["scale"]
    return {"out": y.to(s["q"].dtype), "state": s["state"]}


CHUNK = 64


def _mix_forward(q, k, v, decay, state, lengths, scale):
    """Linear attention in chunks: products within a chunk, states between chunks."""
    batch, length, heads, dk = q.shape
    chunks = -(-length // CHUNK)
    if lengths is not None:
        here = torch.arange(length, device=DEV)[None, :] < lengths[:, None]
        k = torch.where(here[..., None, None], k, 0.0)
        decay = torch.where(here[..., None], decay, 0.0)

    def cut(x):      # [batch, length, heads, ...] -> [batch, heads, chunks, CHUNK, ...]
        pad = [0, 0] * (x.dim() - 2) + [0, chunks * CHUNK - length]
        x = torch.nn.functional.pad(x, pad).unflatten(1, (chunks, CHUNK))
        return x.movedim(3, 1)
    q, k, v, g = cut(q), cut(k), cut(v), cut(decay).double().cumsum(dim=3)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=DEV).tril()
    inside = torch.where(low, g[..., :, None] - g[..., None, :], -math.inf).exp().float()
    total = g[..., -1]
    ends = total.cumsum(dim=2)
    starts = ends - total
    u = (k * (total[..., None] - g).exp().float()[..., None]).transpose(3, 4) @ v
    earlier = torch.ones(chunks, chunks, dtype=torch.bool, device=DEV).tril(-1)
    across = torch.where(earlier, starts[..., :, None] - ends[..., None, :], -math.inf).exp().float()
    before = (across @ u.flatten(3)).unflatten(3, u.shape[3:])
    last = ((ends[..., -1:] - ends).exp().float()[..., None, :] @ u.flatten(3)).unflatten(3, u.shape[3:])[:, :, 0]
    if state is not None:
        before = before + starts.exp().float()[..., None, None] * state[:, :, None]
        last = last + ends[..., -1].exp().float()[..., None, None] * state
    y = ((q @ k.transpose(3, 4)) * inside) @ v + (q @ before) * g.exp().float()[..., None]
    y = y.movedim(1, 3).flatten(1, 2)[:, :length] * scale
    if lengths is not None:
        y = torch.where(here[..., None, None], y, 0.0)
    return y, last


def _mix(s, case):
    dtype = s["q"].dtype
    leaves = _leaves(s)
    x = {n: s[n].detach().float() for n in leaves}
    if case["train"]:
        for t in x.values():
            t.requires_grad_(True)
    y, last = _mix_forward(x["q"], x["k"], x["v"], x["decay"], x.get("state"), s.get("lengths"), s["scale"])
    out = {"out": y.detach().to(dtype), "state": last.detach()}
    if case["train"]:
        ends, gs = ((y, last), (s["g"].float(), s["gs"])) if case["carry"] else ((y,), (s["g"].float(),))
        grads = torch.autograd.grad(ends, [x[n] for n in leaves], gs)
        out.update({"d" + n: t.to(s[n].dtype) for n, t in zip(leaves, grads)})
    return out


def _loss(s, case):
    x, w, targets, eps = s["x"].detach(), s["w"].detach(), s["targets"], case["smooth"]
    xf = x.float()
    wf = (w.t() if case["tied"] else w).float()
    z = xf @ wf
    m = z.amax(dim=1, keepdim=True)
    z = z - m
    here, at = targets >= 0, targets.clamp(min=0)[:, None]
    mean = z.mean(dim=1) if eps else 0.0
    zt = z.gather(1, at)[:, 0]
    e = z.exp_()
    total = e.sum(dim=1, keepdim=True)
    loss = torch.where(here, total.log()[:, 0] - (1 - eps) * zt - eps * mean, 0.0)
    if not case["train"]:
        return (loss,)
    g = torch.where(here, s["g"], 0.0)[:, None]
    d = e.mul_(g / total)
    if eps:
        d -= g * (eps / z.shape[1])
    d.scatter_add_(1, at, g * (eps - 1))
    dw = d.t() @ xf if case["tied"] else xf.t() @ d
    return loss, (d @ wf.t()).to(x.dtype), dw.to(w.dtype)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "embed":
        n, width, vocab = case["n"], case["width"], case["vocab"]
        moved = e * width * (min(n, vocab) + n) + 8 * n
        if case["train"]:
            moved += e * width * (n + vocab)
        return {"bytes": moved, "flops": n * width * (2 if case["train"] else 1)}
    if case["op"] == "loss":
        n, width, vocab = case["n"], case["width"], case["vocab"]
        once = e * width * (n + vocab)
        passes = 3 if case["train"] else 1      # logits, and both gradients' products
        return {"bytes": once * (2 if case["train"] else 1) + 12 * n, "flops": 2 * passes * n * width * vocab}
    heads, dk, dv = case["batch"] * case["heads"], case["dk"], case["dv"]
    if case["op"] == "step":
        return {"bytes": heads * (8 * dk * dv + e * 2 * (dk + dv) + 4), "flops": heads * dk * dv * 5}
    rows, states = heads * case["length"], (2 if case["carry"] else 1)
    moved = rows * (2 * e * (dk + dv) + 4) + 4 * states * heads * dk * dv
    flops = rows * dk * dv * 5
    if case["train"]:
        moved += rows * (2 * e * (dk + dv) + 4) + 4 * (2 if case["carry"] else 0) * heads * dk * dv
        flops *= 3
    return {"bytes": moved, "flops": flops}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _exact_mix(s, case):
    """The recurrence, one token after the other, and back."""
    q, k, v, a = (s[n].detach().double().movedim(1, 0) for n in ("q", "k", "v", "decay"))
    length, batch, heads, dk = q.shape
    live = torch.ones(length, batch, 1, dtype=torch.double, device=DEV)
    if "lengths" in s:
        live = (torch.arange(length, device=DEV)[:, None] < s["lengths"]).double()[..., None]
    a = torch.exp(a * live)[..., None, None]
    q, k, v = (t * live[..., None] for t in (q, k, v))
    S = s["state"].detach().double().clone() if "state" in s else torch.zeros(batch, heads, dk, v.shape[-1], device=DEV).double()
    g = s["g"].double().movedim(1, 0) * live[..., None] * s["scale"] if case["train"] else None
    y, dq = torch.empty_like(v), torch.empty_like(q)
    for t in range(length):
        S.mul_(a[t]).add_(k[t].unsqueeze(3) * v[t].unsqueeze(2))
        y[t] = (q[t].unsqueeze(2) @ S).squeeze(2) * s["scale"]
        if case["train"]:
            dq[t] = (S @ g[t].unsqueeze(3)).squeeze(3)
    out = {"out": y.movedim(0, 1), "state": S}
    if not case["train"]:
        return out
    R = s["gs"].double().clone() if case["carry"] else torch.zeros_like(S)
    ending = (S * R).sum(dim=(2, 3))
    dk_, dv_ = torch.empty_like(q), torch.empty_like(v)
    for t in range(length - 1, -1, -1):
        R.add_(q[t].unsqueeze(3) * g[t].unsqueeze(2))
        dk_[t] = (R @ v[t].unsqueeze(3)).squeeze(3) * live[t][..., None]
        dv_[t] = (k[t].unsqueeze(2) @ R).squeeze(2)
        R.mul_(a[t])
    da = ((q * dq).sum(3) - (k * dk_).sum(3)).flip(0).cumsum(0).flip(0) + ending
    out.update(dq=dq.movedim(0, 1), dk=dk_.movedim(0, 1), dv=dv_.movedim(0, 1), ddecay=(da * live).movedim(0, 1))
    if case["carry"]:
        out["dstate"] = R
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        table, tokens = s["table"].detach().double(), s["tokens"]
        y = table.index_select(0, tokens) * s["scale"]
        if not case["train"]:
            return (y,)
        order = torch.argsort(tokens, stable=True)
        found, count = torch.unique_consecutive(tokens[order], return_counts=True)
        sums = torch.segment_reduce(s["g"].double()[order], "sum", lengths=count, axis=0)
        return y, torch.zeros_like(table).index_copy(0, found, sums * s["scale"])
    if case["op"] == "step":
        S = torch.exp(s["decay"].double())[..., None, None] * s["state"].double()
        S = S + s["k"].double().unsqueeze(3) @ s["v"].double().unsqueeze(2)
        return {"out": (s["q"].double().unsqueeze(2) @ S).squeeze(2) * s["scale"], "state": S}
    if case["op"] == "mix":
        return _exact_mix(s, case)
    x, w, targets, eps = s["x"].detach().double(), s["w"].detach().double(), s["targets"], case["smooth"]
    z = torch.nn.functional.linear(x, w if case["tied"] else w.t())
    vocab = z.shape[1]
    logp = torch.log_softmax(z, dim=1)
    del z
    here, at = targets >= 0, targets.clamp(min=0)[:, None]
    loss = -(1 - eps) * logp.gather(1, at)[:, 0] - eps * logp.mean(1)
    loss = torch.where(here, loss, 0)
    if not case["train"]:
        return (loss,)
    g = torch.where(here, s["g"], 0).double()[:, None]
    d = logp.exp_().sub_(eps / vocab).scatter_add_(1, at, torch.full_like(g, eps - 1)).mul_(g)
    return loss, d @ (w if case["tied"] else w.t()), d.t() @ x if case["tied"] else x.t() @ d
