"""SiLU in 32 bits, relative to its value, however far below 0.  Bounds: the exponential
is good to 2 U, the sum and the reciprocal to 3, the products to one each; where 1 +
x (1 - s) is small, its rounding counts as one of s (1 + |x|)."""
import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lo,hi", [(-80, -40), (-40, -15), (-15, -6), (-6, -2), (-2, 0), (0, 2), (2, 15), (15, 80)])
def test_f32(lo, hi):
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(100 + lo)
    x = torch.rand((4, 20001), generator=gen) * (hi - lo) + lo
    xd = x.cuda().requires_grad_(True)
    y = F.activation(xd, "silu")
    dx, = torch.autograd.grad(y, xd, torch.ones_like(y))
    v = x.double()
    s = 1 / (1 + torch.exp(-v))
    R.close(y, v * s, 8 * R.U * (v * s).abs(), "y")
    R.close(dx, s * (1 + v * (1 - s)), 12 * R.U * s * (1 + v.abs()), "dx")
