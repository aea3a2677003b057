"""layer_norm of segments whose values are all equal: the mean is that value and the
normed values are 0, whatever the value's size.  y is the bias itself, the weight's
gradient 0, and dx = r (a - mean(a)) with r = 1 / sqrt(eps).  A block of equal values
is exact in 8 bits too (its scale is the value), where a row holds whole groups."""
import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
VALUES = [1000.0, 8064.0, 29952.0, -29952.0, 0.1, -1e-3, 123456.789, 3e7, 0.0, 1.0 / 3.0]


def _run(rows, width, groups, blk, dt):
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(rows * 3 + width)
    # neighbouring segments hold other values, where a row may hold several
    n = rows if blk else rows * groups
    v = torch.tensor([VALUES[i % len(VALUES)] for i in range(n)]).to(DT[dt])
    x = v.repeat_interleave(rows * width // n).reshape(rows, width)
    w, b = 1 + 0.2 * torch.randn(width, generator=gen), 0.2 * torch.randn(width, generator=gen)
    dy = torch.randn((rows, width), generator=gen).to(DT[dt])
    args = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = F.layer_norm(*args, eps=EPS, groups=groups, tgrid=(1, blk) if blk else None)
    dx, dw, db = torch.autograd.grad(y, args, dy.cuda())
    assert torch.equal(y.cpu(), b.to(DT[dt]).expand(rows, width))
    assert torch.equal(dw.cpu(), torch.zeros(width))
    D, r = width // groups, EPS ** -0.5
    a = (dy.double() * w.double()).reshape(rows, groups, D)
    size = a.abs() + a.abs().mean(2, keepdim=True)
    want = (r * (a - a.mean(2, keepdim=True))).reshape(rows, width)
    R.close(dx, want, ((64 + D / 64) * R.U * r * size).reshape(rows, width), "dx")
    assert torch.equal(F.layer_norm(x.cuda(), w.cuda(), b.cuda(), eps=EPS, groups=groups), y)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,groups", [
    (10, 1, 1), (10, 7, 1), (10, 96, 1), (20, 100, 1), (10, 1000, 1), (10, 2057, 1), (10, 3000, 1), (10, 4096, 1),
    (10, 4104, 1), (10, 5001, 1), (10, 16384, 1), (10, 13003, 1), (10, 16391, 1), (4, 33000, 1), (2, 300001, 1),
    (30, 640, 10), (30, 144, 3), (12, 4096, 64), (700, 520, 5)])
def test_equal_values(rows, width, groups, dt):
    _run(rows, width, groups, 0, dt)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,groups,blk", [
    (10, 1024, 1, 128), (10, 48, 1, 16), (10, 96 * 2, 1, 32), (10, 256 * 3, 1, 64), (10, 5120, 1, 128), (10, 16384, 1, 128),
    (4, 34816, 1, 128), (10, 2048, 16, 128), (10, 768, 12, 32)])
def test_equal_values_in_8_bits(rows, width, groups, blk, dt):
    _run(rows, width, groups, blk, dt)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("width,groups", [(96, 1), (1000, 1), (4096, 1), (2057, 1), (512, 8), (20000, 1)])
def test_squares_that_overflow(width, groups, dt):
    """Values whose squared deviations are infinite in 32 bits: 1 / sqrt(inf) = 0, the result is the bias and x has
    no gradient, as the same formula gives it in plain 32-bit operations."""
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(width)
    x = (torch.randn((4, width), generator=gen) * 1e30 + 1e29).to(DT[dt])
    w, b = torch.randn(width, generator=gen), torch.randn(width, generator=gen)
    args = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = F.layer_norm(*args, groups=groups)
    assert torch.equal(y.cpu(), b.to(DT[dt]).expand(4, width))
    dx, dw, db = torch.autograd.grad(y, args, torch.randn((4, width), generator=gen).to(DT[dt]).cuda())
    assert not bool(dx.any()) and not bool(dw.any()) and bool(torch.isfinite(db).all())
