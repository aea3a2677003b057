"""functional.activation and its backward pass, with the input kept as it is or
in 8 bits, against the 64-bit forms of tests/row_ref.py."""
import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
KINDS = ("relu2", "silu", "gelu")


def _F():
    from pratchya_amd import functional
    return functional


def _K():
    from pratchya_amd import _kernels
    return _kernels


def _run(x, dy, kind, blk=0):
    xd = x.cuda().requires_grad_(True)
    y = _F().activation(xd, kind, tgrid=(1, blk) if blk else None)
    return (y,) + torch.autograd.grad(y, xd, dy.cuda())


def _check(x, dy, kind, blk=0, what=""):
    want, bound = R.activation(x, kind, dy, blk)
    got = _run(x, dy, kind, blk)
    for g, v, e, n in zip(got, want, bound, ("y", "dx")):
        R.close(g, v, e, f"{what} {kind} {n}")
    return got


def _inputs(rows, width, dt, seed, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    return ((torch.randn((rows, width), generator=gen) * scale).to(DT[dt]),
            torch.randn((rows, width), generator=gen).to(DT[dt]))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 7), (3, 9), (5, 64), (2, 1000), (33, 1023), (1, 4096), (300, 513)])
def test_shapes(rows, width, kind, dt):
    x, dy = _inputs(rows, width, dt, rows + width)
    got = _check(x, dy, kind)
    assert torch.equal(_F().activation(x.cuda(), kind), got[0])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,blk", [
    (1, 16, 16), (3, 1024, 128), (5, 2176, 128), (4, 96, 32), (7, 48, 16), (2, 192, 64), (1000, 128, 128), (9, 384, 128),
    (6, 128, 128), (13, 640, 64), (64, 4096, 128), (3, 32, 32), (1, 64, 64), (511, 16, 16), (2, 8320, 64),
    (1, 128, 128), (2, 256, 128), (4, 256, 128)])
def test_stored_input(rows, width, blk, dt):
    x, dy = _inputs(rows, width, dt, rows + width)
    x[:, ::61] *= 30
    for kind in KINDS:
        _check(x, dy, kind, blk, f"{rows}x{width} blk {blk}")
    y, stored = _K().activation(x.cuda(), "relu2", (1, blk))
    for got, want in zip(stored, _K().quantize(x.cuda(), (1, blk))):
        assert got.shape == want.shape and got.dtype == want.dtype
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_stored_input_edges(dt):
    """The quantizer's rare paths: zeros, values below its clamp, a huge value beside small ones, infinity, NaN
    (their own groups only), rounding midpoints."""
    x, _ = _inputs(12, 1024, "f32", 3, 1.0)
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
    for blk in (16, 32, 64, 128):
        y, stored = _K().activation(x.cuda(), "relu2", (1, blk))
        for got, want in zip(stored, _K().quantize(x.cuda(), (1, blk))):
            a, b = got.view(torch.uint8).cpu(), want.view(torch.uint8).cpu()
            if got.dtype == torch.float32:
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                a, b = got.nan_to_num(7.0).cpu(), want.nan_to_num(7.0).cpu()
            elif got.dtype == torch.float8_e4m3fn:      # a NaN's sign is free
                a, b = torch.where((a & 127) == 127, 127, a), torch.where((b & 127) == 127, 127, b)
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
def test_range(kind):
    """From values whose exponentials vanish or overflow to denormals and signed zeros; NaN stays NaN."""
    v = torch.cat([torch.linspace(-120, 120, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-40, 3e3, -3e3, 1e18]),
                   torch.logspace(-8, 1, 500), -torch.logspace(-8, 1, 500)])[None]
    _check(v, torch.ones_like(v), kind)
    odd = torch.tensor([[1.0, float("nan"), 2.0]])
    y, dx = _run(odd, torch.ones_like(odd), kind)
    assert torch.isnan(y).tolist() == torch.isnan(dx).tolist() == [[False, True, False]]


def test_gradient_by_differences():
    """Central differences of the 64-bit sum of the f32 outputs; second and third derivatives are below 4."""
    gen = torch.Generator().manual_seed(7)
    x, dy = _inputs(3, 200, "f32", 8)
    v = torch.randn(x.shape, generator=gen)
    t = 2.0 ** -7
    for kind in KINDS:
        def f(s):
            return float((_F().activation((x + s * v).cuda(), kind).double().cpu() * dy.double()).sum())
        exact = float((_run(x, dy, kind)[1].double().cpu() * v.double()).sum())
        # relu2's derivative bends at 0: an element there is off by t v^2 at most
        size = (dy.abs() * v.abs() ** 3).sum() * t * t + (dy.abs() * v ** 2 * (x.abs() < t * v.abs())).sum() * t
        allowed = 4 * float(size) + 64 * R.U * float((dy.abs() * (1 + x * x)).sum()) / t
        assert abs((f(t) - f(-t)) / (2 * t) - exact) <= allowed, kind


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strides(dt):
    gen = torch.Generator().manual_seed(21)
    wide = torch.randn((4, 6, 333), generator=gen).to(DT[dt])
    gw = torch.randn((4, 6, 207), generator=gen).to(DT[dt])
    forms = [lambda t: t[..., 33:133], lambda t: t[:, :1, 7:107].expand(4, 6, 100),
             lambda t: t[..., 1:101].transpose(0, 1), lambda t: t[:, ::2, 5:105], lambda t: t[..., 2:202:2],
             lambda t: t[0, 0, 3:103]]
    for fx in forms:
        for fg in forms:
            x, g = fx(wide), fg(gw)
            if x.shape != g.shape:
                continue
            xd = fx(wide.cuda()).detach().requires_grad_(True)
            y = _F().activation(xd, "silu")
            dx, = torch.autograd.grad(y, xd, fg(gw.cuda()))
            want, bound = R.activation(x, "silu", g)
            R.close(y, want[0], bound[0], "y")
            R.close(dx, want[1], bound[1], "dx")


@pytest.mark.parametrize("blk", [16, 128])
def test_strided_stored(blk):
    gen = torch.Generator().manual_seed(22)
    wide = torch.randn((6, 3000), generator=gen).to(torch.bfloat16)
    gw = torch.randn((6, 2500), generator=gen).to(torch.bfloat16)
    for width in (2048, 2176):
        x, dy = wide[:, 5:5 + width], gw[:, 3:3 + width]
        xd = wide.cuda()[:, 5:5 + width].detach().requires_grad_(True)
        y = _F().activation(xd, "gelu", tgrid=(1, blk))
        dx, = torch.autograd.grad(y, xd, gw.cuda()[:, 3:3 + width])
        want, bound = R.activation(x, "gelu", dy, blk)
        R.close(y, want[0], bound[0], "y")
        R.close(dx, want[1], bound[1], "dx")


def test_graph_replays():
    K = _K()
    x, dy = (t.cuda() for t in _inputs(300, 2176, "bf16", 51))

    def work():
        y, q = K.activation(x, "silu", (1, 128))
        return (y, K.activation_bwd(q, dy, "silu", (1, 128)), K.activation(x, "gelu")[0], K.activation_bwd(x, dy, "gelu"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (52, 53, 54):
        for t, v in zip((x, dy), _inputs(300, 2176, "bf16", seed)):
            t.copy_(v)
        want = [t.clone() for t in work()]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, v in zip(out, want):
            assert torch.equal(t, v)


def test_offsets_past_32_bits():
    rows, width = 2 ** 19 + 1, 4096
    x = torch.empty((rows, width), dtype=torch.bfloat16, device="cuda").normal_()
    dy = torch.empty_like(x).normal_()
    y, q = _K().activation(x, "relu2", (1, 128))
    dx = _K().activation_bwd(q, dy, "relu2", (1, 128))
    last = slice(rows - 2, rows)
    want, bound = R.activation(x[last].cpu(), "relu2", dy[last].cpu(), 128)
    R.close(y[last], want[0], bound[0], "y")
    R.close(dx[last], want[1], bound[1], "dx")
    del y, q, dx, dy
    step = 2 ** 31 - 4096
    rows = x.reshape(-1).as_strided((2, 1000), (step, 1))
    want, bound = R.activation(rows.cpu(), "silu")
    R.close(_K().activation(rows, "silu")[0], want[0], bound[0], "y, strided")


def test_empty_and_refusals():
    F, K = _F(), _K()
    for shape in ((0, 64), (3, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        F.activation(x, "silu").sum().backward()
        assert x.grad.shape == x.shape
    x = torch.zeros((0, 64), device="cuda", requires_grad=True)
    F.activation(x, "silu", tgrid=(1, 64)).sum().backward()
    assert x.grad.shape == x.shape
    x = torch.zeros((4, 96), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="unknown activation"):
        F.activation(x, "relu")
    with pytest.raises(RuntimeError, match="GPU only"):
        F.activation(x.detach().cpu())
    with pytest.raises(TypeError, match="float16"):
        F.activation(x.half())
    for tgrid in ((1, 128), (2, 32), (1, 8), (1, 0), (1, 24)):
        with pytest.raises(ValueError, match="block grid"):
            F.activation(x, tgrid=tgrid)
    with pytest.raises(ValueError, match="input"):
        K.activation_bwd(torch.zeros((4, 95), device="cuda"), torch.zeros((4, 96), device="cuda"), "silu")
    with pytest.raises(ValueError, match="input"):
        K.activation_bwd(torch.zeros((4, 96), device="cuda").bfloat16(), torch.zeros((4, 96), device="cuda"), "silu")
    q = K.quantize(x.detach(), (1, 32))
    with pytest.raises(ValueError, match="stored"):
        K.activation_bwd(q, torch.zeros((2, 192), device="cuda"), "silu", (1, 32))
    g, = torch.autograd.grad(F.activation(x, "silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
