"""Plain 64-bit forms of the row operators (layer norm, activations, token log
probabilities) and the error bounds that follow from f32 arithmetic, for their
tests.

Bounds: u = 2^-24.  A sum of n f32 terms in any order is within n u of the sum
of their magnitudes; `N` below covers the additions on the longest path of a
segment's reduction (its length over the lanes, and the tree) and the few
roundings after it.  A result stored in bf16 adds half a bf16 step, 2^-8 of its
magnitude at most."""
import math

import numpy as np
import torch

from oracle import qarr_oracle as O

U = 2.0 ** -24


def stored_values(x: torch.Tensor, blk: int) -> torch.Tensor:
    """What x [rows, width] (CPU) quantized with tgrid (1, blk) stands for, by the oracle, in 64 bits."""
    f = x.float().numpy()
    v = O.dequantize_impl(*O.quantize_impl(f, (1, blk)), "float32", (1, blk))
    return torch.from_numpy(np.array(v, dtype=np.float64).reshape(f.shape))


def layer_norm(x, w, b, eps, groups, dy=None, blk=0):
    """(y, dx, dw, db) and their bounds for f32 results, all [rows, width] / [width] in 64 bits."""
    rows, width = x.shape
    D = width // groups
    u64 = x.double()
    seg = u64.reshape(rows, groups, D)
    mean = seg.mean(2, keepdim=True)
    r = 1 / torch.sqrt(((seg - mean) ** 2).mean(2, keepdim=True) + eps)
    wd = torch.ones(width, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(width, dtype=torch.float64) if b is None else b.double()
    h = ((seg - mean) * r)
    y = h.reshape(rows, width) * wd + bd
    N = 64 + D / 64
    # the mean is off by up to N u mean|x|, the deviation by the square of that and N u of itself
    off = N * U * (1 + r * seg.abs().mean(2, keepdim=True))
    hb = (off * (1 + h.abs())).reshape(rows, width)
    yb = hb * wd.abs() + 4 * U * (y.abs() + bd.abs())
    if dy is None:
        return (y,), (yb,)
    src = (u64 if not blk else stored_values(x, blk)).reshape(rows, groups, D)
    h = (src - mean) * r
    hb = (off * (1 + h.abs())).reshape(rows, width)
    g = dy.double()
    a = (g * wd).reshape(rows, groups, D)
    m1, m2 = a.mean(2, keepdim=True), (a * h).mean(2, keepdim=True)
    dx = (r * (a - m1 - h * m2)).reshape(rows, width)
    mags = a.abs() + a.abs().mean(2, keepdim=True) + h.abs() * (a * h).abs().mean(2, keepdim=True)
    m2b = (a.abs() * off * (1 + h.abs())).mean(2, keepdim=True)
    dxb = (r * (2 * off * mags * (1 + h.abs()) + h.abs() * m2b
                + off * (1 + h.abs()) * (a * h).abs().mean(2, keepdim=True))).reshape(rows, width)
    h = h.reshape(rows, width)
    dw, db = (g * h).sum(0), g.sum(0)
    n = rows + 16
    dwb = (g.abs() * hb).sum(0) + n * U * (g * h).abs().sum(0)
    return (y, dx, dw, db), (yb, dxb, dwb, n * U * g.abs().sum(0))


def activation(x, kind, dy=None, blk=0):
    v = x.double()
    s = v if not blk else stored_values(x, blk)
    phi = torch.exp(-s * s / 2) / math.sqrt(2 * math.pi)
    if kind == "relu2":
        y, d = v.clamp(min=0) ** 2, 2 * s.clamp(min=0)
        yb, db = 4 * U * y, 4 * U * d
    elif kind == "silu":
        p = torch.sigmoid(s)
        y, d = v * torch.sigmoid(v), p * (1 + s * (1 - p))
        # e^x in f32 through a product with log2(e): a relative error of some |x| u
        yb, db = (16 + 4 * v.abs()) * U * y.abs(), (16 + 4 * s.abs()) * U * p * (1 + s.abs())
    else:
        P = torch.special.ndtr(s)
        y, d = v * torch.special.ndtr(v), P + s * phi
        # the distribution function to some steps of 1, the density like silu's exponential
        yb, db = 16 * U * v.abs(), 16 * U + (16 + 4 * s * s) * U * s.abs() * phi
    if dy is None:
        return (y,), (yb,)
    g = dy.double()
    return (y, d * g), (yb, db * g.abs() + 2 * U * (d * g).abs())


def token_logprobs(x, tokens, g=None, gh=None):
    """(logprobs, entropy, dx) and bounds; x [rows, vocab], masked rows and tokens as the operator defines them."""
    u = x.double()
    rows, V = u.shape
    empty = (u == -math.inf).all(1)
    m = u.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    d = u - m
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    logs = torch.where(s == 0, 0.0, torch.log(s))
    lp = d - logs
    p = torch.exp(lp)
    plp = torch.where(p == 0, 0.0, p * lp)
    H = -plp.sum(1)
    t = tokens.clamp(0, V - 1)[:, None]
    out = torch.where(tokens < 0, 0.0, lp.gather(1, t)[:, 0])
    out = torch.where(tokens >= V, math.nan, out)
    # exponentials: some |x| u each; their sum over the lanes and the tree
    N = 64 + V / 128
    size = 8 + d.clamp(min=-1e30).abs().nan_to_num(0)
    sb = (torch.where(p == 0, 0.0, p * size).sum(1) * 4 + N) * U
    lpb = sb + 4 * U * torch.where(tokens < 0, 0.0, lp.gather(1, t)[:, 0].abs().nan_to_num(0, 0, 0) + logs[:, 0].abs())
    Hb = (plp.abs().sum(1) + 1) * (sb + N * U) + 4 * (torch.where(p == 0, 0.0, p * size * (1 + lp.abs())).sum(1) + H.abs()
                                                      + logs[:, 0].abs()) * U
    if g is None and gh is None:
        return (out, H), (lpb, Hb)
    c = torch.where(tokens < 0, 0.0, torch.zeros(rows) if g is None else g.double())[:, None].double()
    ch = torch.zeros(rows, 1).double() if gh is None else gh.double()[:, None]
    dx = -p * c - ch * torch.where(p == 0, 0.0, p * (lp + H[:, None]))
    dx = torch.where(empty[:, None], 0.0, dx)
    here = (tokens >= 0) & (tokens < V)
    one = torch.zeros_like(u)
    one[here] = one[here].scatter(1, t[here], 1.0)
    dx = dx + one * c
    rel = 4 * size * U + sb[:, None] + 16 * U
    mag = p * (c.abs() + ch.abs() * torch.where(p == 0, 0.0, lp.abs() + H.abs()[:, None]))
    # f32 exponentials below 2^-126 are flushed
    dxb = rel * (mag + p * ch.abs()) + p * ch.abs() * Hb[:, None] + 4 * U * one * c.abs() + 2.0 ** -125 * (
        c.abs() + ch.abs() * 200)
    return (out, H, dx), (lpb, Hb, dxb)


def close(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str):
    """got within bound of want plus its own type's rounding; NaN and infinities in the same places."""
    step = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -23
    tiny = 2.0 ** -118      # exponentials below 2^-126 are flushed; times a factor of up to 2^7
    got = got.detach().double().cpu().reshape(want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[odd].nan_to_num(0), want[odd].nan_to_num(0)), f"{what}: infinities differ"
    err = (got - want).abs()[~odd]
    allowed = (bound.expand_as(want) + step * want.abs() + tiny)[~odd]
    bad = err > allowed
    if bool(bad.any()):
        i = int((err / allowed).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound; worst "
                             f"{got[~odd][i]:.9g} for {want[~odd][i]:.9g}, allowed {allowed[i]:.3g}")
