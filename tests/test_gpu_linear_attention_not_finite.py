"""NaN and infinities in functional.linear_attention reach what the recurrence lets them reach:
results of tokens before theirs (gradients of k and v: of tokens behind) keep every bit, and all
are as finite as those of the recurrence in 64 bits."""
import math

import pytest
import torch

from tests import row_ref as R
from tests.test_gpu_linear_attention import DT, _F, make, reference

pytestmark = pytest.mark.gpu

INPUTS = ("q", "k", "v", "g", "state", "dout", "dstate")
RESULTS = ("out", "state", "dq", "dk", "dv", "dg", "dstate")


def call(data):
    q, k, v, g, state, dout, dstate = (t.cuda() for t in data)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, state)]
    r = _F().linear_attention(*leaves[:4], state=leaves[4], scale=0.25)
    got = (r.out, r.state) + torch.autograd.grad((r.out, r.state), leaves, (dout, dstate))
    return {n: t.detach().cpu() for n, t in zip(RESULTS, got)}


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("T,at,D,E", [(70, 37, 64, 64), (150, 20, 48, 80), (40, 31, 7, 33), (600, 577, 16, 16), (90, 50, 128, 128)])
def test_reach(T, at, D, E, where, dt, value):
    data = make(2, T, 2, D, E, DT[dt], seed=T)
    clean = call(data)
    data[INPUTS.index(where)][1, at, 1, 3] = value
    got = call(data)
    want, bound = reference(*data[:5], None, 0.25, *data[5:])
    for name, t in got.items():
        # the other sequence and the other head
        assert torch.equal(t[0], clean[name][0]), name
        other = (1, 0) if name in ("state", "dstate") else (1, slice(None), 0)
        assert torch.equal(t[other], clean[name][other]), name
        if name in ("out", "dq"):
            assert torch.equal(t[1, :at], clean[name][1, :at]), name
        if name in ("dk", "dv"):
            assert torch.equal(t[1, at + 1:], clean[name][1, at + 1:]), name
        if name == "dg" and where in ("k", "v"):
            continue      # a sum over later tokens, it takes in what is not finite there
        fine = torch.isfinite(want[name])
        assert torch.equal(torch.isfinite(t), fine), name
        R.close(t[fine], want[name][fine], bound[name][fine], name)
