"""functional.token_logprobs against the 64-bit form of tests/row_ref.py: log
probabilities, entropy, the best alternatives (exact indices, ties to the lowest)
and the logits' gradient, over vocabularies from 1 up, masks, rows masked
everywhere, infinities and NaN, strides, streams, graphs and refusals."""
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
INF = math.inf


def _F():
    from pratchya_amd import functional
    return functional


def _K():
    from pratchya_amd import _kernels
    return _kernels


def _inputs(rows, vocab, dt, seed, scale=2.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, vocab), generator=gen) * scale).to(DT[dt])
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    return x, tokens, torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)


def _best(x, top):
    """The top indices by value, NaN first, equal values by index."""
    v = x.double()
    nan = torch.isnan(v)
    order = torch.sort(torch.where(nan, INF, v), dim=1, descending=True, stable=True).indices
    first = torch.sort(torch.gather(nan, 1, order).int(), dim=1, descending=True, stable=True).indices
    return torch.gather(order, 1, first)[:, :top]


def _check(x, tokens, g=None, gh=None, top=0, what=""):
    xd = x.cuda().requires_grad_(True)
    r = _F().token_logprobs(xd, tokens.cuda(), entropy=True, top=top)
    want, bound = R.token_logprobs(x, tokens, g, gh)
    R.close(r.logprobs, want[0], bound[0], f"{what} logprobs")
    R.close(r.entropy, want[1], bound[1], f"{what} entropy")
    if top:
        best = _best(x, top)
        assert torch.equal(r.top_tokens.cpu(), best), f"{what}: other alternatives"
        for k in range(top):
            w, b = R.token_logprobs(x, best[:, k])
            R.close(r.top_logprobs[:, k], w[0], b[0], f"{what} alternative {k}")
    if g is not None or gh is not None:
        outs = [(o, c.cuda()) for o, c in ((r.logprobs, g), (r.entropy, gh)) if c is not None]
        dx, = torch.autograd.grad([o for o, _ in outs], xd, [c for _, c in outs])
        assert dx.dtype == x.dtype
        R.close(dx, want[2], bound[2], f"{what} dx")
    # without gradients: the same bits
    n = _F().token_logprobs(x.cuda(), tokens.cuda(), entropy=True, top=top)
    for a, b in zip(r, n):
        assert a is None or torch.equal(a.detach().nan_to_num(9.0), b.nan_to_num(9.0))
    return r


SIZES = [(1, 1), (3, 2), (5, 7), (4, 63), (2, 64), (3, 100), (2, 1000), (2, 4099), (3, 8192), (2, 20001), (2, 50021),
         (3, 65536), (1, 131072), (1, 300001), (300, 511)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_sizes(rows, vocab, dt):
    x, tokens, g, gh = _inputs(rows, vocab, dt, rows + vocab)
    for top in sorted({0, min(vocab, 1), min(vocab, 5), min(vocab, 64)}):
        _check(x, tokens, g, gh, top, f"{rows}x{vocab} top {top}")


@pytest.mark.parametrize("g,gh", [(True, False), (False, True)])
def test_single_cotangents(g, gh):
    x, tokens, a, b = _inputs(9, 3001, "f32", 3)
    _check(x, tokens, a if g else None, b if gh else None)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [5, 100, 4099, 65536])
def test_masks(vocab, dt):
    """A padded vocabulary, rows with one or no unmasked logit, masks of the type's lowest value, tokens that
    are masked, none at all, or beyond the vocabulary."""
    x, tokens, g, gh = _inputs(10, vocab, dt, vocab)
    x[:, vocab - vocab // 3:] = -INF
    tokens %= vocab - vocab // 3
    x[1] = -INF                                            # nothing left
    x[2], x[2, 3] = -INF, 0.5                              # one left
    tokens[2] = 3
    x[3] = -INF
    x[3, 3], tokens[3] = 2.0, 4                            # a masked token
    x[4] = torch.finfo(DT[dt]).min                         # all at the lowest value
    x[5] = torch.finfo(DT[dt]).min
    x[5, 2], tokens[5] = 1.5, 2
    tokens[6], tokens[7] = -1, -100                        # no token
    tokens[8] = vocab                                      # beyond
    x[9, 0], tokens[9] = torch.finfo(DT[dt]).max, 1
    top = min(vocab, 20)
    r = _check(x, tokens, g, gh, top, f"vocab {vocab}")
    assert r.logprobs[1] == -INF and r.entropy[1] == 0 and r.logprobs[6] == 0 and r.logprobs[7] == 0
    assert r.top_tokens[1].tolist() == list(range(top)) and bool((r.top_logprobs[1] == -INF).all())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_nonfinite(dt):
    """NaN or +inf spoil their own row only; NaN ranks above all numbers."""
    x, tokens, g, gh = _inputs(7, 5000, dt, 17)
    x[1, 0] = math.nan
    x[2, 4999] = -math.nan
    x[3, 77] = INF
    x[4] = math.nan
    x[5, 10], x[5, 20], x[5, 30] = INF, math.nan, -INF
    r = _check(x, tokens, g, gh, 12)
    assert torch.isnan(r.logprobs).tolist() == [False, True, True, True, True, True, False]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [63, 64, 2048, 2049, 50021, 65536, 200000])
def test_order_of_alternatives(vocab, dt):
    """Ties and adversarial orders: all equal, two values, rising and falling, the largest ones side by side or
    far apart, signed zeros."""
    idx = torch.arange(vocab).float()
    gen = torch.Generator().manual_seed(1)
    rows = [torch.zeros(vocab), idx % 2, idx % 3 == 1, idx / vocab, -idx / vocab, (idx >= vocab - 70) * (idx - vocab),
            (idx % 1024 == 7) * 3.0, torch.where(idx % 2 == 0, 0.0, -0.0), torch.randint(0, 4, (vocab,), generator=gen),
            (idx < 64) * idx, ((idx // 8) % 256 == 5) * 1.0, torch.where(idx < vocab // 2, -INF, 1.0)]
    x = torch.stack([r.float() for r in rows]).to(DT[dt])
    tokens = torch.zeros(len(rows), dtype=torch.int64)
    for top in (1, 20, 63):
        r = _F().token_logprobs(x.cuda(), tokens.cuda(), top=top)
        assert torch.equal(r.top_tokens.cpu(), _best(x, top)), top


def test_sums_and_far_values():
    """Logits far from zero, a token sure to come, and a row's gradients that sum to zero."""
    for scale, shift in ((1.0, 1e4), (1.0, -3e4), (40.0, 0.0), (1e-3, 0.0)):
        x, tokens, g, gh = _inputs(6, 2003, "f32", 23, scale)
        _check(x + shift, tokens, g, gh, 5, f"{scale} {shift}")
    x, tokens, g, gh = _inputs(4, 999, "f32", 24)
    x[torch.arange(4), tokens] += 60
    _check(x, tokens, g, gh, 3, "sure")
    xd = x.cuda().requires_grad_(True)
    r = _F().token_logprobs(xd, tokens.cuda())
    assert r.entropy is None and r.top_tokens is None
    dx, = torch.autograd.grad(r.logprobs, xd, g.cuda())
    assert float(dx.double().sum(1).abs().max()) <= 2000 * R.U * float(g.abs().max()) * 2


def test_gradient_by_differences():
    """Central differences of log probabilities and entropies; their third derivatives along a unit-scale
    direction are below 100."""
    x, tokens, g, gh = _inputs(4, 60, "f32", 31)
    gen = torch.Generator().manual_seed(32)
    v = torch.randn(x.shape, generator=gen)
    xd = x.cuda().requires_grad_(True)
    r = _F().token_logprobs(xd, tokens.cuda(), entropy=True)
    dx, = torch.autograd.grad((r.logprobs, r.entropy), xd, (g.cuda(), gh.cuda()))
    t = 2.0 ** -7

    def f(s):
        r = _F().token_logprobs((x + s * v).cuda(), tokens.cuda(), entropy=True)
        return float((r.logprobs.double().cpu() * g).sum() + (r.entropy.double().cpu() * gh).sum())
    size = float(g.abs().sum() + gh.abs().sum())
    allowed = size * (t * t / 6 * 100 + 256 * R.U * 10 / t)
    exact = float((dx.double().cpu() * v.double()).sum())
    assert abs((f(t) - f(-t)) / (2 * t) - exact) <= allowed


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strides(dt):
    """Logits as a slice at an odd address, of a wider array, transposed, broadcast, with leading axes; tokens in
    32 bits and strided; cotangents broadcast."""
    gen = torch.Generator().manual_seed(41)
    wide = torch.randn((4, 6, 1333), generator=gen).to(DT[dt])
    for f in (lambda t: t[..., 33:1133], lambda t: t[..., 1:1101].transpose(0, 1),
              lambda t: t[:, :1, 7:1107].expand(4, 6, 1100), lambda t: t[..., 2:1202:2], lambda t: t[2, 3, 1:]):
        x = f(wide)
        lead = x.shape[:-1]
        tok = torch.randint(0, x.shape[-1], lead + (2,), generator=gen)
        g = torch.randn(lead, generator=gen)
        xd = f(wide.cuda()).detach().requires_grad_(True)
        r = _F().token_logprobs(xd, tok.cuda().int()[..., 1], entropy=True, top=4)
        flat = x.reshape(-1, x.shape[-1])
        want, bound = R.token_logprobs(flat, tok[..., 1].reshape(-1), g.reshape(-1), torch.full((flat.shape[0],), 0.5))
        assert r.logprobs.shape == lead and r.top_tokens.shape == lead + (4,)
        R.close(r.logprobs.reshape(-1), want[0], bound[0], "logprobs")
        assert torch.equal(r.top_tokens.reshape(-1, 4).cpu(), _best(flat, 4))
        dx, = torch.autograd.grad((r.logprobs, r.entropy), xd, (g.cuda(), torch.tensor(0.5).cuda().expand(lead)))
        R.close(dx.reshape(flat.shape), want[2], bound[2], "dx")


def test_repeats_and_streams():
    x, tokens, g, gh = (t.cuda() for t in _inputs(64, 30001, "bf16", 51))
    K = _K()

    def work():
        out = K.token_logprobs(x, tokens, True, 20, True)
        return out + (K.token_logprobs_bwd(x, tokens, out[4], g, gh),)
    first = work()
    _F().token_logprobs(*(t.cuda() for t in _inputs(3, 77, "f32", 52)[:2]), top=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = work()
    side.synchronize()
    for a, b, c in zip(first, work(), again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replays():
    x, tokens, g, gh = (t.cuda() for t in _inputs(40, 9001, "f32", 61))
    K = _K()

    def work():
        out = K.token_logprobs(x, tokens, True, 7, True)
        return out + (K.token_logprobs_bwd(x, tokens, out[4], g, gh),)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (62, 63, 64):
        for t, v in zip((x, tokens, g, gh), _inputs(40, 9001, "f32", seed)):
            t.copy_(v)
        want = [t.clone() for t in work()]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, v in zip(out, want):
            assert torch.equal(t, v)


def test_offsets_past_32_bits():
    """Rows of logits 2^31 elements apart, and a gradient of more than 2^31 elements."""
    step = 2 ** 31 + 24
    buf = torch.zeros(step + 5000, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((2, 4001), (step, 1))
    v, tokens, g, gh = _inputs(2, 4001, "bf16", 71)
    x.copy_(v)
    want, bound = R.token_logprobs(v, tokens, g, gh)
    out = _K().token_logprobs(x, tokens.cuda(), True, 9, True)
    R.close(out[0], want[0], bound[0], "logprobs")
    assert torch.equal(out[3].cpu(), _best(v, 9))
    dx = _K().token_logprobs_bwd(x, tokens.cuda(), out[4], g.cuda(), gh.cuda())
    R.close(dx, want[2], bound[2], "dx")
    del x, buf, dx
    rows, vocab = 2 ** 15 + 1, 65536
    x = torch.empty((rows, vocab), dtype=torch.bfloat16, device="cuda").normal_()
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    g = torch.randn(rows, device="cuda")
    out = _K().token_logprobs(x, tokens, False, 0, True)
    dx = _K().token_logprobs_bwd(x, tokens, out[4], g, None)
    last = slice(rows - 2, rows)
    want, bound = R.token_logprobs(x[last].cpu(), tokens[last].cpu(), g[last].cpu(), None)
    R.close(out[0][last], want[0], bound[0], "logprobs")
    R.close(dx[last], want[2], bound[2], "dx")


def test_empty_and_refusals():
    F, K = _F(), _K()
    x = torch.zeros((0, 50), device="cuda", requires_grad=True)
    r = F.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), True, 3)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 3)
    r.logprobs.sum().backward()
    assert x.grad.shape == x.shape
    x = torch.zeros((4, 50), device="cuda", requires_grad=True)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="GPU only"):
        F.token_logprobs(x.detach().cpu(), t.cpu())
    with pytest.raises(TypeError, match="float16"):
        F.token_logprobs(x.half(), t)
    with pytest.raises(TypeError, match="int64"):
        F.token_logprobs(x, t.float())
    with pytest.raises(ValueError, match="tokens"):
        F.token_logprobs(x, t[:3])
    for top in (-1, 51, 65):
        with pytest.raises(ValueError, match="alternatives"):
            F.token_logprobs(x, t, top=top)
    with pytest.raises(ValueError, match="alternatives"):
        F.token_logprobs(torch.zeros((4, 0), device="cuda"), t)
    r = F.token_logprobs(x, t, top=2)
    assert not r.top_logprobs.requires_grad
    g, = torch.autograd.grad(r.logprobs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    st = torch.zeros((4, 3), device="cuda")
    with pytest.raises(ValueError, match="cotangent"):
        K.token_logprobs_bwd(x.detach(), t, st, torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError, match="statistics"):
        K.token_logprobs_bwd(x.detach(), t, st[:3])
