"""functional.linear_cross_entropy from 256 rows on, where the logits stay in the products'
tiles: edge tiles that overlap their neighbours, targets on both sides of every tile's
and wave's border, pieces of the vocabulary in the backward pass, slices of K, rows and
weights inside larger arrays, rows of NaN.  References and bounds are those of
test_gpu_linear_cross_entropy.py."""
import math

import pytest
import torch

from tests import row_ref as R
from tests.test_gpu_linear_cross_entropy import DT, _F, _check, _normal

pytestmark = pytest.mark.gpu


def _targets(n, V, seed):
    """Random ones, and the columns on both sides of the tiles' borders."""
    t = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed))
    marks = [c for b in (0, 128, 256, 384, 512, V - 256, V - 128, V // 64 * 64, V) for c in (b - 1, b) if 0 <= c < V]
    t[:len(marks)] = torch.tensor(marks)
    t[len(marks):len(marks) + 3] = torch.tensor([-1, -7, -(1 << 62)])
    t[n - 1] = V - 1
    return t


SIZES = [(256, 256, 256), (257, 300, 257), (300, 777, 320), (511, 1025, 260), (333, 4099, 449), (1000, 700, 512)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,V,C", SIZES)
def test_edges(n, V, C, tied, dt):
    x, w = _normal((n, C), DT[dt], n), _normal((C, V), DT[dt], V, 2.0 / math.sqrt(C))
    for a in (0.0, 0.2):
        _check(x, w, _targets(n, V, n), a, _normal((n,), torch.float32, V), tied)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,V,C,dt", [(1000, 16384, 1024, "bf16"), (1000, 4100, 1000, "f32"), (1000, 16384, 1000, "f32")])
def test_slices_of_the_vocabulary_as_k(n, V, C, dt, tied):
    """Few tiles of the gradient of x: K, the vocabulary, in slices joined at the end."""
    x, w = _normal((n, C), DT[dt], 1), _normal((C, V), DT[dt], 2, 2.0 / math.sqrt(C))
    _check(x, w, _targets(n, V, 3), 0.0, _normal((n,), torch.float32, 4), tied)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("V,dt", [(40011, "bf16"), (65536, "bf16"), (23000, "f32")])
def test_pieces_of_gradients(V, dt, tied):
    n, C = 8192, 256
    x, w = _normal((n, C), DT[dt], 1), _normal((C, V), DT[dt], 2, 0.2)
    _check(x, w, _targets(n, V, 3), 0.1 if V == 40011 else 0.0, _normal((n,), torch.float32, 4), tied)


@pytest.mark.parametrize("tied", [False, True])
def test_inside_larger_arrays(tied):
    """Operands read as they lie: what surrounds them is NaN."""
    F = _F()
    n, V, C = 320, 640, 256
    x, w = _normal((n, C), DT["bf16"], 1), _normal((C, V), DT["bf16"], 2, 0.2)
    targets, g = _targets(n, V, 3), _normal((n,), torch.float32, 4)
    want = _check(x, w, targets, 0.1, g, tied)
    for before, behind in ((0, 64), (8, 8), (3, 5)):
        X = torch.full((n + 2, C + before + behind), math.nan, dtype=DT["bf16"], device="cuda")
        xs = X[1:n + 1, before:before + C]
        xs.copy_(x.cuda())
        ws = w.t() if tied else w
        W = torch.full((ws.shape[0] + 2, ws.shape[1] + before + behind), math.nan, dtype=DT["bf16"], device="cuda")
        wv = W[1:ws.shape[0] + 1, before:before + ws.shape[1]]
        wv.copy_(ws.cuda())
        xs, wv = xs.detach().requires_grad_(True), wv.detach().requires_grad_(True)
        y = F.linear_cross_entropy(xs, wv.t() if tied else wv, targets.cuda(), label_smoothing=0.1)
        got = (y,) + torch.autograd.grad(y, (xs, wv), g.cuda())
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (before, behind)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rows_apart(dt):
    """A row of NaN spoils its own loss and gradient alone; rows without a target or with a cotangent of 0 train nothing."""
    F = _F()
    n, V, C = 300, 512, 256
    x, w = _normal((n, C), DT[dt], 1), _normal((C, V), DT[dt], 2, 0.2)
    targets = _targets(n, V, 3)
    y0, dx0, _ = _check(x, w, targets, 0.0, torch.ones(n), False)
    bad = x.clone()
    bad[77, 5] = math.nan
    xd, wd = bad.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = F.linear_cross_entropy(xd, wd, targets.cuda())
    dx, = torch.autograd.grad(y, xd, torch.ones(n, device="cuda"))
    keep = torch.arange(n, device="cuda") != 77
    assert bool(torch.isnan(y[77])) and bool(torch.isnan(dx[77]).all())
    assert torch.equal(y[keep], y0[keep]) and torch.equal(dx[keep], dx0[keep])
    none = torch.full((n,), -1, device="cuda")
    xd = x.cuda().requires_grad_(True)
    y = F.linear_cross_entropy(xd, wd, none, label_smoothing=0.1)
    dx, dw = torch.autograd.grad(y, (xd, wd), torch.full((n,), 1e30, device="cuda"))
    assert not bool(y.any()) and not bool(dx.any()) and not bool(dw.any())
    y = F.linear_cross_entropy(xd, wd, targets.cuda())
    dx, dw = torch.autograd.grad(y, (xd, wd), torch.zeros(n, device="cuda"))
    assert not bool(dx.any()) and not bool(dw.any())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,V,C", [(40, 100, 64), (64, 1024, 256), (300, 512, 256), (512, 1024, 320)])
@pytest.mark.parametrize("tied", [False, True])
def test_padding_that_is_not_finite(n, V, C, tied, dt):
    """Rows without a target may hold anything: no loss, no gradient of theirs, none of the weight from them."""
    F = _F()
    x, w = _normal((n, C), DT[dt], 1), _normal((C, V), DT[dt], 2, 0.2)
    targets = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(3))
    rows = torch.tensor([0, 3, 17, n - 1])
    targets[rows] = -1
    g = _normal((n,), torch.float32, 4)
    want = _check(x, w, targets, 0.1, g, tied)
    bad = x.clone()
    bad[rows[0]], bad[rows[1], 2], bad[rows[2]], bad[rows[3], C - 1] = math.nan, math.inf, -math.inf, math.nan
    g[rows[1]] = math.nan
    xd, wd = bad.cuda().requires_grad_(True), (w.t().contiguous() if tied else w).cuda().requires_grad_(True)
    y = F.linear_cross_entropy(xd, wd.t() if tied else wd, targets.cuda(), label_smoothing=0.1)
    got = (y,) + torch.autograd.grad(y, (xd, wd), g.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_near_and_far():
    """Losses near 0 keep the digits of the others' sum; logits of +-1000 do not overflow."""
    F = _F()
    n, V, C = 256, 512, 256
    x = torch.zeros((n, C))
    x[:, 0] = 1.0
    w = torch.zeros((C, V))
    w[0, 300], w[0, 5] = 1000.0, -1000.0
    targets = torch.full((n,), 300)
    targets[1], targets[2] = 5, 7
    for dt in DT.values():
        xd, wd = x.to(dt).cuda().requires_grad_(True), w.to(dt).cuda()
        y = F.linear_cross_entropy(xd, wd, targets.cuda())
        dx, = torch.autograd.grad(y.sum(), xd)
        assert y[:3].tolist() == [0.0, 2000.0, 1000.0] and bool(torch.isfinite(dx).all())
        assert dx[:3, 0].tolist() == [0.0, 2000.0, 1000.0]
    w[0, 300] = 14.0
    few = math.log1p((V - 2) * math.exp(-14.0))
    y = F.linear_cross_entropy(x.cuda(), w.cuda(), targets.cuda())[0].double()
    assert abs(float(y) - few) <= 64 * R.U * few


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,V,C,dt,smooth", [(300, 33100, 640, "f32", 0.1), (1000, 17000, 1027, "f32", 0.0),
                                             (260, 33024, 512, "f32", 0.0), (513, 22016, 3136, "bf16", 0.1)])
def test_last_round_of_tiles(n, V, C, dt, smooth, tied):
    """One or a few tiles more than the chip computes at once: the vocabulary's end goes another way."""
    x, w = _normal((n, C), DT[dt], 1), _normal((C, V), DT[dt], 2, 2.0 / math.sqrt(C))
    targets = _targets(n, V, 3)
    main = 256 // -(-n // 256) * 256
    targets[40:48] = torch.tensor([main - 257, main - 256, main - 1, main, main + 1, main + 63, V - 65, V - 64])
    _check(x, w, targets, smooth, _normal((n,), torch.float32, 4), tied)


@pytest.mark.parametrize("n,V,C", [(100, 2000, 256), (600, 4096, 512)])
@pytest.mark.parametrize("smooth", [0.0, 0.1])
def test_one_cotangent_for_all(n, V, C, smooth):
    """A mean's cotangent, the same for all rows and halfway between two bf16 values: its rounding must
    not stand in every row.  What is left of a gradient's error is its own rounding, 2^-8 / sqrt(3) of
    its norm at most (uniform in half a step), and the logits' gradients', which is random and mostly in
    their small values: together below sqrt(2) of it; the cotangent's own would be 2^-8."""
    from tests.test_gpu_linear_cross_entropy import reference
    F = _F()
    x, w = _normal((n, C), DT["bf16"], 1), _normal((C, V), DT["bf16"], 2, 1.0 / math.sqrt(C))
    targets = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(3))
    g = torch.full((n,), (1 + 2.0 ** -8) / (1 - smooth) / 512)
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    got = torch.autograd.grad(F.linear_cross_entropy(xd, wd, targets.cuda(), label_smoothing=smooth), (xd, wd), g.cuda())
    want, _ = reference(x, w, targets, smooth, g)
    for a, b in zip(got, want[1:]):
        assert float((a.double().cpu() - b).norm() / b.norm()) < 2.0 ** -8 * math.sqrt(2 / 3)
