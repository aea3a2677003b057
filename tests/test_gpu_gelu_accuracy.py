"""GELU in 32 bits, relative to its value.  Bounds: x / sqrt 2 carries a rounding of
x's and one of the constant's, and a relative change of z changes erfc(z) by at most
2 z^2 + 1 = x^2 + 1 times as much; erfc itself is good to 8 U, the products to a few.
So P(x) is within (12 + 2 x^2) U of itself.  The density's exponent x^2 / 2 is rounded
twice: (12 + 2 x^2) U of it too."""
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

RANGES = [(-12, -6), (-6, -4), (-4, -2), (-2, -0.5), (-0.5, 0.5), (0.5, 2), (2, 4), (4, 12)]


@pytest.mark.parametrize("lo,hi", RANGES)
def test_f32(lo, hi):
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(int(100 + 2 * lo))
    x = torch.rand((4, 20001), generator=gen) * (hi - lo) + lo
    xd = x.cuda().requires_grad_(True)
    y = F.activation(xd, "gelu")
    dx, = torch.autograd.grad(y, xd, torch.ones_like(y))
    v = x.double()
    P, p = torch.erfc(v * -math.sqrt(0.5)) / 2, torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    rel = (12 + 2 * v * v) * R.U
    R.close(y, v * P, rel * v.abs() * P, "y")
    R.close(dx, P + v * p, rel * (P + v.abs() * p), "dx")
