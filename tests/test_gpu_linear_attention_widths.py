"""functional.linear_attention at widths and layouts that choose its ways of reading:
whole vectors through buffers (also of widths that no tile has), odd widths whose last
vector is moved, arrays inside larger ones, rows too far apart for 32-bit offsets, many
heads and few (segments and their parts), calls on several streams at once.  References and
bounds are those of test_gpu_linear_attention.py."""
import math

import pytest
import torch

from tests import row_ref as R
from tests.test_gpu_linear_attention import DT, U, _F, check, make, reference

pytestmark = pytest.mark.gpu

WIDTHS = [(48, 80), (72, 24), (8, 120), (4, 12), (57, 101), (9, 15), (15, 64), (64, 127), (7, 3), (128, 33)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,E", WIDTHS)
def test_widths(D, E, dt):
    """Two sequences of several segments, one of them padded from the middle of a chunk on."""
    T = 620
    q, k, v, g, state, dout, dstate = make(2, T, 2, D, E, DT[dt], seed=D)
    lengths = torch.tensor([T, 401])
    for t in (q, k, v, g, dout):
        t[1, 401:] = math.nan
    check(q, k, v, g, state, lengths, D ** -0.5, dout, dstate)
    check(q, k, v, g, None, lengths, D ** -0.5, dout, None)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("before,behind", [(8, 8), (16, 0), (1, 2)])
@pytest.mark.parametrize("D,E", [(64, 64), (48, 80), (57, 33)])
def test_inside_larger_arrays(D, E, before, behind, dt):
    """What lies before, behind and between the rows is NaN."""
    F = _F()
    B, T, H = 2, 300, 2
    q, k, v, g, state, dout, dstate = make(B, T, H, D, E, DT[dt], seed=D)

    def inside(t):
        wide = torch.full((B, T + 2, H, t.shape[-1] + before + behind), math.nan, dtype=t.dtype, device="cuda")
        view = wide[:, 1:T + 1, :, before:before + t.shape[-1]]
        view.copy_(t.cuda())
        return view.detach()
    leaves = [inside(t).requires_grad_(True) for t in (q, k, v)] + [g.cuda().requires_grad_(True), state.cuda().requires_grad_(True)]
    r = F.linear_attention(*leaves[:4], state=leaves[4], scale=0.2)
    got = torch.autograd.grad((r.out, r.state), leaves, (inside(dout), dstate.cuda()))
    want, bound = reference(q, k, v, g, state, None, 0.2, dout, dstate)
    for name, t in zip(("out", "state", "dq", "dk", "dv", "dg", "dstate"), (r.out, r.state) + got):
        R.close(t, want[name], bound[name], name)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,H,D,E", [(1, 2500, 1, 16, 16), (1, 1100, 7, 16, 32), (1, 600, 2, 128, 128), (3, 300, 200, 8, 8)])
def test_segments(B, T, H, D, E, dt):
    """From one head, whose segments are the shortest, to more heads than the chip holds workgroups of."""
    q, k, v, g, state, dout, dstate = make(B, T, H, D, E, DT[dt], seed=T)
    check(q, k, v, g, state, None, D ** -0.5, dout, dstate)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_segments_without_gradients(dt):
    """Without a backward pass to come a sequence of these sizes is cut into more segments: other
    roundings, the same bounds."""
    F = _F()
    B, T, H, D, E = 6, 1040, 50, 16, 16
    q, k, v, g, state, dout, dstate = make(B, T, H, D, E, DT[dt], seed=T)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g, state)]
    r = F.linear_attention(*leaves[:4], state=leaves[4], scale=0.25)
    got = (r.out, r.state) + torch.autograd.grad((r.out, r.state), leaves, (dout.cuda(), dstate.cuda()))
    with torch.no_grad():
        plain = F.linear_attention(*leaves[:4], state=leaves[4], scale=0.25)
    want, bound = reference(q, k, v, g, state, None, 0.25, dout, dstate)
    for name, t in zip(("out", "state", "dq", "dk", "dv", "dg", "dstate", "out", "state"), got + tuple(plain)):
        R.close(t, want[name], bound[name], name)


def test_slow_decays_over_segments():
    """A decay's gradient sums over all that follows: tokens thousands apart, hardly forgotten."""
    q, k, v, g, state, dout, dstate = make(1, 3000, 1, 32, 32, torch.float32, seed=2)
    check(q, k, v, 1e-3 * g, state, None, 0.2, dout, dstate)
    check(q, k, v, (1e-3 * g).bfloat16(), state, torch.tensor([2222]), 0.2, dout, dstate)


def test_rows_far_apart():
    """Rows beyond 32-bit offsets give what the same rows side by side give, within a rounding of
    the type (another order of nothing but instructions)."""
    F = _F()
    T, D, step = 66000, 64, 16384 + 64
    gen = torch.Generator(device="cuda").manual_seed(1)
    far = torch.empty(T * step, dtype=torch.bfloat16, device="cuda")
    assert far.numel() * 2 > 1 << 31
    rows = [far[i * D:].as_strided((1, T, 1, D), (T * step, step, step, 1)) for i in range(4)]
    near = [torch.randn((1, T, 1, D), generator=gen, device="cuda").bfloat16() for _ in range(4)]
    for a, b in zip(rows, near):
        a.copy_(b)
    g = -0.1 * torch.rand((1, T, 1), generator=gen, device="cuda")
    res = []
    for q, k, v, dout in (rows, near):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, g)]
        r = F.linear_attention(*leaves, scale=0.125)
        res.append((r.out.detach(), r.state.detach()) + torch.autograd.grad(r.out, leaves, dout))
    for a, b in zip(*res):
        a, b = a.double(), b.double()
        assert bool(torch.isfinite(a).all())
        assert float((a - b).abs().max()) <= 2.0 ** -7 * float(b.abs().max())


def test_one_token_of_many():
    """A batch of single tokens through linear_attention agrees with the step in place."""
    F = _F()
    for dt in DT.values():
        q, k, v, g, state, _, _ = (t.cuda() for t in make(300, 1, 5, 64, 48, dt, seed=3))
        r = F.linear_attention(q, k, v, g, state=state, scale=0.5)
        s = state.clone()
        y = F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s, scale=0.5)
        R.close(r.state, s.double().cpu(), 8 * U * (state.abs().cpu() + 40).double(), "state")
        half = 2.0 ** -7 if dt == torch.bfloat16 else 0.0
        size = (q.double().abs().transpose(-1, -2)[:, 0].movedim(-1, 1)[..., None] * s.double().abs()).sum(-2)
        R.close(r.out[:, 0], y.double().cpu(), ((half + 300 * U) * 0.5 * size).cpu(), "out")


def test_calls_at_once():
    """Two streams' calls share nothing but their inputs."""
    F = _F()
    q, k, v, g, state, dout, dstate = (t.cuda() for t in make(2, 900, 8, 64, 64, torch.bfloat16, seed=5))
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, state)]

    def work():
        r = F.linear_attention(*leaves[:4], state=leaves[4], scale=0.125)
        return (r.out, r.state) + torch.autograd.grad((r.out, r.state), leaves, (dout, dstate))
    want = [t.detach().clone() for t in work()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for w in got:
        assert all(torch.equal(a.detach(), b) for a, b in zip(w, want))
