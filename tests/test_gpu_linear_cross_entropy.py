"""functional.linear_cross_entropy and its gradients against 64 bits: sizes that no tile
divides, both layouts of the weight, several pieces of the vocabulary, targets that
stand for nothing, label smoothing, cotangents, layouts, streams, graphs.

Bounds (u = 2^-24).  A logit is a sum of C products, exact ones of bf16 values; of f32
values six products of pieces each, what they leave out below 2^-22 of the product: in
any order within (6 C + 64) u sum |x w| + 2^-22 sum |x w|.  e^d is within (16 + 4 |d|) u,
a sum over the vocabulary adds V / 256 + 64 roundings on its longest path.  A gradient
of a logit in bf16 is rounded once (2^-8); the gradients are sums of n or V such."""
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
U = R.U


def _F():
    from pratchya_amd import functional
    return functional


def _normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def reference(x, w, targets, a, g=None):
    """(loss, dx, dw) and their bounds in 64 bits on the GPU; x [n, C], w [C, V]."""
    bf = x.dtype == torch.bfloat16
    u, v = x.cuda().double(), w.cuda().double()
    n, C = u.shape
    V = v.shape[1]
    targets = targets.cuda()
    z, size = u @ v, u.abs() @ v.abs()
    zb = ((6 * C + 64) * U + (0 if bf else 2.0 ** -22)) * size
    m = z.amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    d = (z - m).abs()
    sumb = ((p * (zb + (16 + 4 * d) * U)).sum(1, keepdim=True) + (V / 256 + 64) * U)
    lseb = sumb + 4 * U * (lse.abs() + m.abs())
    t = targets.clamp(0, V - 1)[:, None]
    zt, ztb = z.gather(1, t), zb.gather(1, t)
    loss = (1 - a) * (lse - zt) + a * (lse - z.mean(1, keepdim=True))
    lossb = lseb + ztb + 4 * U * (zt.abs() + m.abs()) + a * (zb.mean(1, keepdim=True)
                                                             + (V / 256 + 64) * U * z.abs().mean(1, keepdim=True))
    loss, lossb = loss[:, 0], lossb[:, 0] + 4 * U * loss[:, 0].abs()
    loss = torch.where(targets < 0, 0.0, loss)
    loss = torch.where(targets >= V, math.nan, loss)
    if g is None:
        return loss.cpu(), lossb.cpu()
    g = torch.where(targets < 0, 0.0, g.cuda().double())[:, None]
    one = torch.zeros_like(z)
    here = (targets >= 0) & (targets < V)
    one[here] = one[here].scatter(1, t[here], 1.0 - a)
    dz = g * (p - one - a / V)
    dzb = g.abs() * (p * (zb + lseb + (24 + 4 * d) * U) + 4 * U * (p + one + a / V) + 2.0 ** -126)
    dzb = dzb + (2.0 ** -8 if bf else 4 * U) * dz.abs()
    dx, dw = dz @ v.t(), u.t() @ dz
    dxb = dzb @ v.abs().t() + ((6 * V + 64) * U + 2.0 ** -22) * (dz.abs() @ v.abs().t())
    dwb = u.abs().t() @ dzb + ((6 * n + 64) * U + 2.0 ** -22) * (u.abs().t() @ dz.abs())
    return (loss.cpu(), dx.cpu(), dw.cpu()), (lossb.cpu(), dxb.cpu(), dwb.cpu())


def _check(x, w, targets, a, g, tied):
    """Loss and gradients of x, w (CPU) with the weight in one of its layouts."""
    F = _F()
    xd = x.cuda().requires_grad_(True)
    leaf = (w.t().contiguous() if tied else w).cuda().requires_grad_(True)
    y = F.linear_cross_entropy(xd, leaf.t() if tied else leaf, targets.cuda(), label_smoothing=a)
    assert y.dtype == torch.float32 and y.shape == targets.shape
    dx, dw = torch.autograd.grad(y, (xd, leaf), g.cuda())
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dw.shape == leaf.shape and dw.is_contiguous()
    want, bound = reference(x.reshape(-1, x.shape[-1]), w, targets.reshape(-1), a, g.reshape(-1))
    R.close(y.reshape(-1), want[0], bound[0], "loss")
    R.close(dx.reshape(want[1].shape), want[1], bound[1], "dx")
    R.close(dw.t() if tied else dw, want[2], bound[2], "dw")
    plain = F.linear_cross_entropy(xd.detach(), leaf.detach().t() if tied else leaf.detach(), targets.cuda(), a)
    assert not plain.requires_grad and torch.equal(plain.nan_to_num(7), y.detach().nan_to_num(7))
    return y, dx, dw


SIZES = [(1, 1, 1), (1, 2, 64), (3, 7, 5), (2, 64, 64), (31, 100, 72), (32, 128, 128), (33, 130, 64), (64, 1000, 256),
         (100, 4099, 65), (130, 513, 200), (128, 2048, 192), (257, 777, 1027), (300, 8192, 64), (512, 1024, 512),
         (256, 4096, 320), (1000, 1280, 128)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,V,C", SIZES)
def test_values_and_gradients(n, V, C, tied, dt):
    x, w = _normal((n, C), DT[dt], n + C), _normal((C, V), DT[dt], V, 2.0 / math.sqrt(C))
    gen = torch.Generator().manual_seed(n)
    targets = torch.randint(0, V, (n,), generator=gen)
    if n > 4:
        targets[1], targets[n - 1], targets[2], targets[4] = -1, -(1 << 40), V - 1, 0
    for a in (0.0, 0.1):
        _check(x, w, targets, a, torch.randn(n, generator=gen) / n, tied)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("tied", [False, True])
def test_pieces(tied, dt):
    """A vocabulary in several pieces, the last one ragged, and one of a whole number of tiles."""
    for n, V, C in ((8192, 20011, 64), (8192, 24576, 64)):
        x, w = _normal((n, C), DT[dt], 1), _normal((C, V), DT[dt], 2, 0.3)
        targets = torch.randint(-1, V, (n,), generator=torch.Generator().manual_seed(3))
        _check(x, w, targets, 0.0, _normal((n,), torch.float32, 4), tied)


def test_targets_beyond():
    """No logit stands for them: NaN, and the gradient of the other terms."""
    x, w = _normal((8, 64), torch.bfloat16, 1), _normal((64, 128), torch.bfloat16, 2)
    targets = torch.tensor([3, 128, 127, 1 << 40, -1, 0, 129, 5])
    y, _, _ = _check(x, w, targets, 0.1, _normal((8,), torch.float32, 3), False)
    assert torch.isnan(y.cpu()).tolist() == [False, True, False, True, False, False, True, False]


@pytest.mark.parametrize("n,V,C", [(4, 100, 64), (300, 1024, 128)])
def test_near_zero(n, V, C):
    """A loss near 0 keeps the digits of the others' sum; a hopeless one does not overflow."""
    F = _F()
    x = torch.zeros((n, C))
    x[:, 0] = 1.0
    w = torch.zeros((C, V))
    w[0, 3], w[0, 5] = 14.0, -900.0
    targets = torch.full((n,), 3)
    targets[1] = 5
    y = F.linear_cross_entropy(x.cuda(), w.cuda(), targets.cuda()).cpu().double()
    few = math.log1p((V - 2) * math.exp(-14.0))
    lse = 14.0 + few
    assert abs(y[0] - few) <= 64 * U * few and abs(y[1] - (lse + 900.0)) <= 8 * U * 914
    yb = F.linear_cross_entropy(x.bfloat16().cuda(), w.bfloat16().cuda(), targets.cuda()).cpu().double()
    assert abs(yb[0] - few) <= 128 * U * few and abs(yb[1] - (lse + 900.0)) <= 8 * U * 914     # 900 = 225 * 4: a bf16 value


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layouts(dt):
    """x and the weight as slices of wider arrays, x of more axes, int32 targets, broadcast cotangents."""
    F = _F()
    wide, big = _normal((6, 10, 200), DT[dt], 1).cuda(), _normal((150, 1000), DT[dt], 2, 0.2).cuda()
    x, w = wide[..., 20:148].requires_grad_(True), big[7:135, 100:612].requires_grad_(True)
    targets = torch.randint(0, 512, (6, 10), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    for weight in (w, w.t().contiguous().t(), w[:, ::2][:, :200], w.t()[100:300].t()):
        t = targets % weight.shape[1]
        for g in (torch.ones((), device="cuda").expand(6, 10), _normal((10, 6), torch.float32, 5).cuda().t()):
            y = F.linear_cross_entropy(x, weight, t.cuda())
            dx, dw = torch.autograd.grad(y, (x, weight), g)
            want, bound = reference(x.detach().reshape(60, 128).cpu(), weight.detach().cpu(), t.reshape(-1),
                                    0.0, g.cpu().reshape(-1))
            R.close(y.reshape(-1), want[0], bound[0], "loss")
            R.close(dx.reshape(60, 128), want[1], bound[1], "dx")
            R.close(dw, want[2], bound[2], "dw")
    one = F.linear_cross_entropy(x[0, 0], w, torch.tensor(3, device="cuda"))
    assert one.shape == ()


def test_one_gradient_alone():
    F = _F()
    x, w = _normal((100, 128), torch.bfloat16, 1).cuda(), _normal((128, 640), torch.bfloat16, 2).cuda()
    t, g = torch.arange(100, device="cuda"), _normal((100,), torch.float32, 3).cuda()
    both = [v.clone().requires_grad_(True) for v in (x, w)]
    want = torch.autograd.grad(F.linear_cross_entropy(*both, t), both, g)
    xa = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(F.linear_cross_entropy(xa, w, t), xa, g)[0], want[0])
    wa = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(F.linear_cross_entropy(x, wa, t), wa, g)[0], want[1])


def test_empty():
    F = _F()
    x = torch.zeros((0, 3, 16), device="cuda", requires_grad=True)
    w = torch.ones((16, 40), device="cuda", requires_grad=True)
    y = F.linear_cross_entropy(x, w, torch.zeros((0, 3), dtype=torch.int64, device="cuda"))
    assert y.shape == (0, 3)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and not bool(dw.any())


@pytest.mark.parametrize("n,V,C", [(200, 1000, 100), (512, 2048, 256)])
def test_same_bits_streams_and_graphs(n, V, C):
    F = _F()
    x, w = (_normal(s, torch.bfloat16, i, 0.3).cuda().requires_grad_(True) for i, s in enumerate(((n, C), (C, V))))
    t, g = torch.randint(0, V, (n,), device="cuda"), _normal((n,), torch.float32, 3).cuda()

    def work():
        y = F.linear_cross_entropy(x, w, t, 0.05)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), g)
    want = [v.clone() for v in work()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(work(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for rep in range(3):
        with torch.no_grad():
            x.copy_(_normal((n, C), torch.bfloat16, 10 + rep))
            t.copy_(torch.randint(-1, V, (n,), device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, work())), rep


def test_changed_input_and_freed_graph():
    F = _F()
    x = _normal((4, 64), torch.bfloat16, 1).cuda().requires_grad_(True)
    w = _normal((64, 128), torch.bfloat16, 2).cuda().requires_grad_(True)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    h = x * 1
    y = F.linear_cross_entropy(h, w, t)
    with torch.no_grad():
        h += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = F.linear_cross_entropy(x, w, t)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()


def test_refusals():
    F = _F()
    x, w = torch.zeros((4, 8), device="cuda"), torch.zeros((8, 20), device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad, error in ((lambda: F.linear_cross_entropy(x, w.bfloat16(), t), TypeError),
                       (lambda: F.linear_cross_entropy(x.half(), w.half(), t), TypeError),
                       (lambda: F.linear_cross_entropy(x, w.t(), t), ValueError),
                       (lambda: F.linear_cross_entropy(x, w[0], t), ValueError),
                       (lambda: F.linear_cross_entropy(x, w[:, :0], t), ValueError),
                       (lambda: F.linear_cross_entropy(x, w, t[:3]), ValueError),
                       (lambda: F.linear_cross_entropy(x, w, t.float()), TypeError),
                       (lambda: F.linear_cross_entropy(x, w, t, -0.1), ValueError),
                       (lambda: F.linear_cross_entropy(x, w, t, 1.5), ValueError),
                       (lambda: F.linear_cross_entropy(x, w, t, float("nan")), ValueError),
                       (lambda: F.linear_cross_entropy(x, w.cpu(), t), RuntimeError),
                       (lambda: F.linear_cross_entropy(x, w, t.cpu()), RuntimeError)):
        with pytest.raises(error):
            bad()
    xg = x.clone().requires_grad_(True)
    d, = torch.autograd.grad(F.linear_cross_entropy(xg, w, t).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        d.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        F.linear_cross_entropy(fwd.make_dual(x, torch.ones_like(x)), w, t)
