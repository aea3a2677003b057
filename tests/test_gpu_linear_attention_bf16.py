"""functional.linear_attention in bf16: arithmetic between its inputs and results as f32 has it.

Bounds.  The inputs are exact, so a result is its own rounding, 2^-8 of itself, off what the
same call in f32 bounds (tests/test_gpu_linear_attention.py), but for the scores and the states
that outputs read, which have two bf16 pieces: 2^-16 of each term, of which an output sums two
kinds with magnitudes A, so 2^-16 A, and as much again for f32's own 16 + 4 |d| units in e^d."""
import pytest
import torch

from tests import row_ref as R
from tests.test_gpu_linear_attention import _F, make, reference

pytestmark = pytest.mark.gpu

NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dstate")


def bounds(q, k, v, g, state, lengths, scale, dout, dstate):
    want, bound = reference(q.float(), k.float(), v.float(), g, state, lengths, scale, dout.float(), dstate)
    mag = reference(*(t.float().abs() for t in (q, k, v)), g, None if state is None else state.abs(), lengths, abs(scale),
                    dout.float().abs(), None if dstate is None else dstate.abs())[0]
    for n in ("out", "dq", "dk", "dv"):
        bound[n] = bound[n] + 2.0 ** -15 * mag[n]      # R.close adds the result's rounding
    return want, bound


@pytest.mark.parametrize("carry", [False, True])
@pytest.mark.parametrize("gates", ["any", "none", "resets"])
@pytest.mark.parametrize("B,T,H,D,E", [(1, 130, 2, 64, 64), (2, 300, 2, 128, 64), (1, 600, 2, 48, 80), (1, 200, 1, 57, 101),
                                       (1, 1100, 1, 128, 128)])
def test_one_rounding(B, T, H, D, E, gates, carry):
    F = _F()
    q, k, v, g, state, dout, dstate = make(B, T, H, D, E, torch.bfloat16, seed=T + D, gates=gates)
    if not carry:
        state = dstate = None
    want, bound = bounds(q, k, v, g, state, None, 0.25, dout, dstate)
    for decays in (True, False):      # a gradient of the decays does not decide what the others hold
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)] + [g.cuda().requires_grad_(decays)]
        s0 = None if state is None else state.cuda().requires_grad_(True)
        r = F.linear_attention(*leaves, state=s0, scale=0.25)
        ends, gs = ((r.out, r.state), (dout.cuda(), dstate.cuda())) if carry else ((r.out,), (dout.cuda(),))
        wrt = leaves[:4 if decays else 3] + ([s0] if carry else [])
        got = torch.autograd.grad(ends, wrt, gs)
        names = NAMES[:2] + NAMES[2:6 if decays else 5] + (("dstate",) if carry else ())
        for name, t in zip(names, (r.out, r.state) + got):
            R.close(t, want[name], bound[name], name)
    with torch.no_grad():
        plain = F.linear_attention(*leaves, state=s0, scale=0.25)
    R.close(plain.out, want["out"], bound["out"], "out without gradients")
    R.close(plain.state, want["state"], bound["state"], "state without gradients")
