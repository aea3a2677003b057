"""functional.layer_norm and its gradients against the 64-bit forms of
tests/row_ref.py: widths from 1 up, odd ones, heads, both types, strided and
broadcast rows, parameters left out, inputs kept in 8 bits (quantized bytes by
the oracle), values far from zero, infinities and NaN in single segments,
offsets past 32 bits, streams, graphs and refusals."""
import numpy as np
import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def _F():
    from pratchya_amd import functional
    return functional


def _K():
    from pratchya_amd import _kernels
    return _kernels


def _inputs(rows, width, dt, seed, w=torch.float32, b=torch.float32, mean=0.3, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, width), generator=gen) * std + mean).to(DT[dt])
    dy = torch.randn((rows, width), generator=gen).to(DT[dt])
    ws = (1 + 0.2 * torch.randn(width, generator=gen)).to(w) if w else None
    bs = (0.2 * torch.randn(width, generator=gen)).to(b) if b else None
    return x, ws, bs, dy


def _grads(x, w, b, dy, groups=1, tgrid=None, eps=EPS):
    """(y, dx, dw, db) through autograd on the GPU."""
    args = [None if t is None else t.detach().cuda().requires_grad_(True) for t in (x, w, b)]
    y = _F().layer_norm(*args, eps=eps, groups=groups, tgrid=tgrid)
    got = iter(torch.autograd.grad(y, [t for t in args if t is not None], dy.cuda()))
    return (y,) + tuple(None if t is None else next(got) for t in args)


def _check(x, w, b, dy, groups=1, blk=0, eps=EPS, what=""):
    got = _grads(x, w, b, dy, groups, (1, blk) if blk else None, eps)
    want, bound = R.layer_norm(x, w, b, eps, groups, dy, blk)
    for g, v, e, n in zip(got, want, bound, ("y", "dx", "dw", "db")):
        if g is not None:
            R.close(g, v, e, f"{what} {n}")
    return got


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,groups", [
    (1, 1, 1), (1, 8, 1), (3, 7, 1), (2, 9, 1), (5, 64, 1), (33, 96, 3), (17, 1000, 1), (4, 2057, 1), (9, 4096, 64),
    (2, 4104, 1), (7, 8192, 1), (3, 16384, 1), (2, 16391, 1), (2, 33000, 1), (300, 256, 1), (1000, 64, 1),
    (70, 1320, 40), (21, 1530, 10), (5, 6, 6), (129, 2048, 16), (3, 512, 1), (600, 1024, 1), (1537, 48, 2),
    (4, 12288, 3), (2, 70000, 2), (1, 4096, 1), (2, 640, 5), (11, 8200, 1)])
def test_shapes(rows, width, groups, dt):
    x, w, b, dy = _inputs(rows, width, dt, rows * 7 + width)
    _check(x, w, b, dy, groups, what=f"{rows}x{width}/{groups}")
    # without gradients: the same values
    y = _F().layer_norm(x.cuda(), w.cuda(), b.cuda(), groups=groups)
    want, bound = R.layer_norm(x, w, b, EPS, groups)
    R.close(y, want[0], bound[0], "no gradients")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("w,b", [(None, None), (torch.float32, None), (None, torch.bfloat16),
                                 (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
def test_parameters(w, b, dt):
    for rows, width, groups in ((37, 520, 1), (50, 256, 4), (6, 4096, 1)):
        x, ws, bs, dy = _inputs(rows, width, dt, 5, w, b)
        got = _check(x, ws, bs, dy, groups, what=f"{w} {b}")
        assert ws is None or got[2].dtype == w
        assert bs is None or got[3].dtype == b


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True),
                                  (False, True, True), (True, False, True)])
@pytest.mark.parametrize("blk", [0, 32])
def test_single_gradients(need, blk):
    """Only some of x, weight and bias ask for a gradient: the others' bits do not change with it."""
    x, w, b, dy = _inputs(40, 768, "bf16", 9)
    full = _grads(x, w, b, dy, tgrid=(1, blk) if blk else None)
    args = [t.cuda().requires_grad_(n) for t, n in zip((x, w, b), need)]
    y = _F().layer_norm(*args, tgrid=(1, blk) if blk else None)
    y.backward(dy.cuda())
    for t, n, v in zip(args, need, full[1:]):
        assert (t.grad is not None) == n
        assert not n or torch.equal(t.grad, v)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,blk,groups", [
    (3, 1024, 128, 1), (5, 2176, 128, 1), (4, 96, 32, 1), (7, 48, 16, 1), (2, 192, 64, 1), (16, 4096, 128, 1),
    (500, 128, 128, 1), (9, 16, 16, 1), (5, 8192, 128, 1), (3, 16384, 64, 1), (2, 17408, 128, 1), (12, 2048, 32, 1),
    (6, 512, 16, 8), (10, 1024, 128, 16), (2, 34816, 128, 1), (1, 128, 128, 1), (300, 1024, 16, 1),
    (4, 6144, 64, 1)])
def test_stored_input(rows, width, blk, groups, dt):
    x, w, b, dy = _inputs(rows, width, dt, rows + width)
    x[:, ::97] *= 30
    x[0, :blk] = 0                                       # a block of zeros
    _check(x, w, b, dy, groups, blk, what=f"{rows}x{width} blk {blk}")
    # the stored form is the quantizer's, byte for byte
    y, st, stored = _K().layer_norm(x.cuda(), w.cuda(), b.cuda(), EPS, groups, True, (1, blk))
    for got, want in zip(stored, _K().quantize(x.cuda(), (1, blk))):
        assert got.shape == want.shape and got.dtype == want.dtype
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_stored_input_edges(dt):
    """Rows whose stored form takes the quantizer's rare paths: all zeros, values below its clamp, a huge
    value beside small ones, an infinity and a NaN (their own rows only), rounding midpoints."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((12, 1024), generator=gen)
    x[0] = 0
    x[1] *= 1e-9
    x[2, 5] = 1e30
    x[3] *= 1e-38
    x[4, 1000] = float("inf")
    x[5, 17] = float("nan")
    x[6] = torch.arange(1024).float() / 64 + 1.0 / 512
    x[7, 512:] = 0
    x[8] *= 1e36
    x = x.to(DT[dt])
    w = torch.ones(1024)
    for blk in (16, 32, 64, 128):
        y, st, stored = _K().layer_norm(x.cuda(), w.cuda(), None, EPS, 1, True, (1, blk))
        for got, want in zip(stored, _K().quantize(x.cuda(), (1, blk))):
            a, b = got.view(torch.uint8).cpu(), want.view(torch.uint8).cpu()
            if got.dtype == torch.float32:
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                a, b = got.nan_to_num(7.0).cpu(), want.nan_to_num(7.0).cpu()
            elif got.dtype == torch.float8_e4m3fn:      # a NaN's sign is free
                a, b = torch.where((a & 127) == 127, 127, a), torch.where((b & 127) == 127, 127, b)
            assert torch.equal(a, b)
        keep = [0, 1, 6, 7, 9, 10, 11]
        want, bound = R.layer_norm(x[keep], w, None, EPS, 1)
        R.close(y[keep], want[0], bound[0], f"finite rows, blk {blk}")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strides(dt):
    """Rows as a slice of a wider array, broadcast rows, transposed arrays, three leading axes, odd addresses."""
    gen = torch.Generator().manual_seed(21)
    w, b = torch.randn(100, generator=gen), torch.randn(100, generator=gen)
    wide = torch.randn((4, 6, 333), generator=gen).to(DT[dt])
    gw = torch.randn((4, 6, 207), generator=gen).to(DT[dt])
    forms = [lambda t: t[..., 33:133], lambda t: t[:, :1, 7:107].expand(4, 6, 100),
             lambda t: t[..., 1:101].transpose(0, 1), lambda t: t[:, ::2, 5:105], lambda t: t[..., 2:202:2]]
    for fx in forms:
        for fg in forms:
            x, g = fx(wide), fg(gw)
            if x.shape != g.shape:
                continue
            xd, gd = fx(wide.cuda()).detach().requires_grad_(True), fg(gw.cuda())
            for blk in (0,):
                y = _F().layer_norm(xd, w.cuda(), b.cuda())
                dx, = torch.autograd.grad(y, xd, gd)
                want, bound = R.layer_norm(x.reshape(-1, 100), w, b, EPS, 1, g.reshape(-1, 100))
                R.close(y.reshape(-1, 100), want[0], bound[0], "y")
                R.close(dx.reshape(-1, 100), want[1], bound[1], "dx")
    # the sum's cotangent is one value broadcast over the array
    x = torch.randn((5, 64), generator=gen).to(DT[dt])
    xd = x.cuda().requires_grad_(True)
    _F().layer_norm(xd, w[:64].cuda()).float().sum().backward()
    want, bound = R.layer_norm(x, w[:64], None, EPS, 1, torch.ones(5, 64))
    R.close(xd.grad, want[1], bound[1], "dx of the sum")


@pytest.mark.parametrize("blk", [16, 128])
def test_strided_stored(blk):
    gen = torch.Generator().manual_seed(22)
    wide = torch.randn((6, 3000), generator=gen).to(torch.bfloat16)
    x, dy = wide[:, 5:2053], torch.randn((6, 2048), generator=gen).to(torch.bfloat16)
    xd = wide.cuda()[:, 5:2053].detach().requires_grad_(True)
    y = _F().layer_norm(xd, tgrid=(1, blk))
    dx, = torch.autograd.grad(y, xd, dy.cuda())
    want, bound = R.layer_norm(x, None, None, EPS, 1, dy, blk)
    R.close(y, want[0], bound[0], "y")
    R.close(dx, want[1], bound[1], "dx")


def test_far_from_zero_and_constant():
    for mean, std in ((1e4, 1.0), (-3e5, 10.0), (0.0, 1e-6), (1e-20, 0.0), (0.1, 0.0), (7.0, 0.0)):
        for width, groups in ((96, 1), (3000, 1), (512, 8)):
            x, w, b, dy = _inputs(6, width, "f32", 11, mean=mean, std=std)
            _check(x, w, b, dy, groups, what=f"mean {mean} std {std}")
    x, w, b, dy = _inputs(5, 300, "bf16", 12)
    _check(x, w, b, dy, eps=0.25, what="eps")


@pytest.mark.parametrize("width,groups", [(256, 4), (4096, 1), (1000, 1)])
def test_nonfinite_segments(width, groups):
    """An infinity or NaN spoils its own segment and its columns' parameter gradients only."""
    x, w, b, dy = _inputs(12, width, "f32", 13)
    bad = x.clone()
    bad[3, 1], bad[7, width - 1] = float("inf"), float("nan")
    y, dx, dw, db = _grads(bad, w, b, dy, groups)
    want, bound = R.layer_norm(x, w, b, EPS, groups, dy)
    D = width // groups
    spoilt = torch.zeros((12, width), dtype=torch.bool)
    spoilt[3, :D] = True
    spoilt[7, width - D:] = True
    assert torch.isnan(y.cpu()[spoilt]).all() and torch.isnan(dx.cpu()[spoilt]).all()
    for g, v, e in ((y, want[0], bound[0]), (dx, want[1], bound[1])):
        R.close(torch.where(spoilt, 0.0, g.cpu()), torch.where(spoilt, 0.0, v), e, "other segments")
    R.close(db, want[3], bound[3], "db")


def test_gradient_by_differences():
    """Directional derivatives of a weighted sum of outputs, by central differences of the 64-bit sum of the
    f32 outputs: the step's third-order term and the outputs' rounding over the step bound the distance."""
    gen = torch.Generator().manual_seed(31)
    for rows, width, groups in ((4, 96, 1), (3, 120, 5)):
        x, w, b, dy = _inputs(rows, width, "f32", 31)
        grads = _grads(x, w, b, dy, groups)[1:]
        t = 2.0 ** -7
        for i, (p, g) in enumerate(zip((x, w, b), grads)):
            v = torch.randn(p.shape, generator=gen)

            def f(s):
                args = [q + s * v if j == i else q for j, q in enumerate((x, w, b))]
                y = _F().layer_norm(*(a.cuda() for a in args), groups=groups)
                return float((y.double().cpu() * dy.double()).sum())
            slope = (f(t) - f(-t)) / (2 * t)
            exact = float((g.double().cpu() * v.double()).sum())
            # third derivatives of a unit-scale norm along a unit-scale direction: below 60 per output
            allowed = t * t / 6 * 60 * float(dy.abs().sum()) + 8 * R.U * float(dy.abs().sum()) * 4 / t
            assert abs(slope - exact) <= allowed, (i, slope, exact, allowed)


def test_repeats_and_streams():
    """The same bits again, on another stream than the current one, and between other work."""
    x, w, b, dy = _inputs(3000, 1024, "bf16", 41)
    first = _grads(x, w, b, dy, tgrid=(1, 128))
    _grads(*_inputs(77, 999, "f32", 42))
    for t, u in zip(first, _grads(x, w, b, dy, tgrid=(1, 128))):
        assert torch.equal(t, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _grads(x, w, b, dy, tgrid=(1, 128))
    side.synchronize()
    for t, u in zip(first, again):
        assert torch.equal(t, u)


def test_graph_replays():
    x, w, b, dy = (t.cuda() for t in _inputs(200, 2048, "bf16", 51))
    K = _K()

    def work():
        y, st, q = K.layer_norm(x, w, b, EPS, 1, True, (1, 128))
        y2, st2, q2 = K.layer_norm(x, w, b, EPS, 32, True, (1, 32))
        return (y, *K.layer_norm_bwd(q, dy, w, st, 1, (1, 128)), y2, *K.layer_norm_bwd(x, dy, w, st2, 32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (52, 53, 54):
        nx, nw, nb, ndy = _inputs(200, 2048, "bf16", seed)
        for t, v in ((x, nx), (w, nw), (b, nb), (dy, ndy)):
            t.copy_(v)
        want = [t.clone() for t in work()]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, v in zip(out, want):
            assert torch.equal(t, v)


def test_offsets_past_32_bits():
    """Rows 2^31 elements apart, and a result of more than 2^31 elements."""
    step = 2 ** 31 + 24
    buf = torch.zeros(step + 5000, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((2, 3000), (step, 1))
    v, w, b, dy = _inputs(2, 3000, "bf16", 61)
    x.copy_(v)
    want, bound = R.layer_norm(v, w, b, EPS, 1, dy)
    y, st, _ = _K().layer_norm(x, w.cuda(), b.cuda(), EPS, 1, True)
    R.close(y, want[0], bound[0], "y")
    dx, dw, db = _K().layer_norm_bwd(x, dy.cuda(), w.cuda(), st)
    R.close(dx, want[1], bound[1], "dx")
    R.close(dw, want[2], bound[2], "dw")
    del x, buf
    rows, width = 2 ** 19 + 1, 4096
    x = torch.empty((rows, width), dtype=torch.bfloat16, device="cuda").normal_()
    dy = torch.empty_like(x).normal_()
    w = torch.randn(width, device="cuda")
    y, st, q = _K().layer_norm(x, w, None, EPS, 1, True, (1, 128))
    dx = _K().layer_norm_bwd(q, dy, w, st, 1, (1, 128), (True, False, False))[0]
    last = slice(rows - 2, rows)
    want, bound = R.layer_norm(x[last].cpu(), w.cpu(), None, EPS, 1, dy[last].cpu(), 128)
    R.close(y[last], want[0], bound[0], "y")
    R.close(dx[last], want[1], bound[1], "dx")


def test_empty():
    F = _F()
    for shape in ((0, 64), (3, 0), (0, 5, 128)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y = F.layer_norm(x, w)
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape and torch.equal(w.grad, torch.zeros_like(w))
    x = torch.zeros((0, 128), device="cuda", requires_grad=True)
    F.layer_norm(x, tgrid=(1, 128)).sum().backward()
    assert x.grad.shape == x.shape


def test_refusals():
    F, K = _F(), _K()
    x = torch.zeros((4, 96), device="cuda")
    with pytest.raises(RuntimeError, match="GPU only"):
        F.layer_norm(x.cpu())
    with pytest.raises(TypeError, match="float16"):
        F.layer_norm(x.half())
    with pytest.raises(TypeError, match="float64"):
        F.layer_norm(x, torch.ones(96, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="groups"):
        F.layer_norm(x, groups=5)
    with pytest.raises(ValueError, match="groups"):
        F.layer_norm(x, groups=0)
    with pytest.raises(ValueError, match="weight"):
        F.layer_norm(x, torch.ones(95, device="cuda"))
    with pytest.raises(ValueError, match="weight"):
        F.layer_norm(x, torch.ones(96))
    with pytest.raises(ValueError, match="contiguous"):
        F.layer_norm(x, None, torch.ones(192, device="cuda")[::2])
    x.requires_grad_(True)
    for tgrid in ((1, 128), (2, 32), (1, 8), (1, 0), (1, 24)):
        with pytest.raises(ValueError, match="block grid"):
            F.layer_norm(x, tgrid=tgrid)
    y = F.layer_norm(x)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    st = torch.zeros((4, 2), device="cuda")
    with pytest.raises(ValueError, match="statistics"):
        K.layer_norm_bwd(x.detach(), torch.zeros((5, 96), device="cuda"), None, st)
    with pytest.raises(ValueError, match="input"):
        K.layer_norm_bwd(torch.zeros((4, 95), device="cuda"), torch.zeros((4, 96), device="cuda"), None, st)
    q = K.quantize(x.detach(), (1, 32))
    with pytest.raises(ValueError, match="stored"):
        K.layer_norm_bwd(q, torch.zeros((2, 192), device="cuda"), None, torch.zeros((2, 2), device="cuda"), 1, (1, 32))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,groups", [
    (70, 1025, 1), (33, 1536, 1), (21, 1537, 1), (40, 2048, 1), (19, 2049, 1), (9, 4097, 1), (30, 5120, 1),
    (5, 6144, 1), (7, 6151, 1), (37, 3300, 3), (11, 5002, 2), (6, 8190, 6), (13, 9, 1), (13, 15, 1), (50, 30, 2)])
def test_teams(rows, width, groups, dt):
    """Segments around the sizes at which teams grow, and ones that end inside a vector."""
    x, w, b, dy = _inputs(rows, width, dt, rows * 11 + width, w=torch.bfloat16)
    _check(x, w, b, dy, groups, what=f"{rows}x{width}/{groups}")


@pytest.mark.parametrize("rows,width,groups,blk", [(4100, 4097, 1, 0), (8200, 2050, 1, 0), (16390, 1029, 1, 0),
                                                   (8193, 2058, 2, 0), (4097, 4160, 1, 32)])
def test_many_rows(rows, width, groups, blk):
    """Rows enough for the backward pass's largest grids."""
    x, w, b, dy = _inputs(rows, width, "bf16", rows + width)
    _check(x, w, b, dy, groups, blk, what=f"{rows}x{width}/{groups}")


def test_an_odd_end_and_its_neighbours():
    """The vector moved back to a segment's end reads and writes nothing outside the segment: what lies
    around it is NaN going in and untouched coming out, and infinities stay in their segment."""
    for dt in (torch.bfloat16, torch.float32):
        for D in (9, 13, 65, 67, 1027, 4097, 16391):
            gen = torch.Generator().manual_seed(D)
            big = torch.full((6, 3 * D), float("nan"), dtype=dt)
            big[1:5, D:2 * D] = torch.randn((4, D), generator=gen).to(dt)
            x, dy = big.cuda()[1:5, D:2 * D], torch.randn((4, D), generator=gen).to(dt)
            y = _F().layer_norm(x)
            want, bound = R.layer_norm(x.cpu(), None, None, EPS, 1)
            R.close(y, want[0], bound[0], f"{dt} {D}")
            x = x.detach().requires_grad_(True)
            (dx,) = torch.autograd.grad(_F().layer_norm(x), x, dy.cuda())
            want, bound = R.layer_norm(x.detach().cpu(), None, None, EPS, 1, dy)
            R.close(dx, want[1], bound[1], f"{dt} {D}")
            three = torch.randn((4, 3 * D), generator=gen).to(dt)
            three[2, D - 1] = float("inf")
            y3 = _F().layer_norm(three.cuda(), groups=3).float().cpu()
            assert torch.isfinite(y3[2, D:]).all() and torch.isfinite(y3[[0, 1, 3]]).all()
            assert not torch.isfinite(y3[2, :D]).any()
