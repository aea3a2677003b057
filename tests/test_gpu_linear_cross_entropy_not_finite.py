"""A row of x that is not finite keeps to itself in functional.linear_cross_entropy: the other rows'
losses and gradients keep every bit, its own loss is NaN or infinite, as its gradient, and the
weight's gradient is not finite unless the row has no target."""
import math

import pytest
import torch

from tests.test_gpu_linear_cross_entropy import DT, _F, _normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,V,C", [(100, 1000, 256), (300, 1024, 320), (300, 777, 257)])
def test_one_row(n, V, C, tied, dt, value):
    F = _F()
    x, w = _normal((n, C), DT[dt], 1).cuda(), _normal((C, V), DT[dt], 2, 0.2).cuda()
    leaf = (w.t().contiguous() if tied else w).requires_grad_(True)
    t, g = torch.arange(n, device="cuda") * 7 % V, _normal((n,), torch.float32, 3).cuda()

    def call(x, t):
        x = x.clone().requires_grad_(True)
        y = F.linear_cross_entropy(x, leaf.t() if tied else leaf, t)
        return (y.detach(),) + torch.autograd.grad(y, (x, leaf), g)
    at = 77
    rest = [i for i in range(n) if i != at]
    bad = x.clone()
    bad[at, 5] = value
    clean, got = call(x, t), call(bad, t)
    for a, b in zip(clean[:2], got[:2]):
        assert torch.equal(a[rest], b[rest])
    assert not math.isfinite(got[0][at]) and not bool(torch.isfinite(got[1][at]).any())
    assert not bool(torch.isfinite(got[2]).any())
    t = t.clone()
    t[at] = -1
    clean, got = call(x, t), call(bad, t)
    assert all(torch.equal(a, b) for a, b in zip(clean, got))
