"""functional.embedding and its table's gradient against plain 64-bit sums: sizes that
no vector divides, tokens that come once, never, a tile's length of times and thousands
of times, tokens that stand for nothing, layouts, streams, graphs.

Bounds (u = 2^-24): a looked-up value is one f32 product; a gradient's sum of m f32
terms in any order is within m u of the sum of their magnitudes, and one product."""
import ctypes

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _F():
    from pratchya_amd import functional
    return functional


def _normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _tokens(kind, n, vocab, seed=7):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randint(0, vocab, (n,), generator=gen)
    if kind == "one":
        t[:] = vocab - 1
    elif kind == "runs":                 # rows of 63, 64, 65, 128, 129 and 200 tokens among others
        at = 0
        for i, m in enumerate((63, 64, 65, 128, 129, 200)):
            t[at:at + m] = (i * 31) % vocab
            at += m
        t = t[torch.randperm(n, generator=gen)]
    elif kind == "none":
        t[torch.rand(n, generator=gen) < 0.3] = -1
        t[::17] = -(1 << 40)
        t[::13] = vocab
        t[::29] = 1 << 40
    elif kind == "sorted":
        t = t.sort().values
    return t


def _check(table, tokens, dy, scale, y, d):
    """y and the gradient d against 64 bits, on the CPU."""
    vocab = table.shape[0]
    flat, g = tokens.reshape(-1), dy.double().reshape(-1, table.shape[1])
    here = (flat >= 0) & (flat < vocab)
    want = table.double()[flat.clamp(0, vocab - 1)] * scale
    want[flat < 0] = 0
    want[flat >= vocab] = float("nan")
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    slack = abs(s32 - scale) / max(abs(scale), 1e-30) + R.U
    R.close(y, want.reshape(y.shape), want.nan_to_num(0).abs().reshape(y.shape) * slack, "y")
    if d is None:
        return
    total, size = torch.zeros(table.shape).double(), torch.zeros(table.shape).double()
    total.index_add_(0, flat[here], g[here])
    size.index_add_(0, flat[here], g[here].abs())
    count = torch.zeros(vocab).double().index_add_(0, flat[here], torch.ones(int(here.sum())).double())
    R.close(d, total * scale, abs(scale) * size * (count[:, None] * R.U + slack + R.U), "dtable")
    assert bool((d.cpu()[count == 0] == 0).all())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("kind,n,vocab,width", [
    ("any", 1, 1, 1), ("any", 3, 5, 7), ("any", 64, 100, 33), ("one", 65, 3, 64), ("one", 64, 3, 64), ("any", 1000, 700, 129),
    ("runs", 1500, 513, 257), ("runs", 700, 40, 1031), ("none", 777, 97, 520), ("sorted", 5000, 1000, 64),
    ("any", 40, 70001, 24), ("one", 9001, 2, 40), ("any", 4097, 131, 2057), ("none", 2000, 1, 9)])
def test_values_and_gradient(kind, n, vocab, width, dt):
    F = _F()
    table, tokens, dy = _normal((vocab, width), DT[dt], 1), _tokens(kind, n, vocab), _normal((n, width), DT[dt], 2)
    for scale in (1.0, 45.25483399593904):
        w = table.cuda().requires_grad_(True)
        y = F.embedding(w, tokens.cuda(), scale=scale)
        d, = torch.autograd.grad(y, w, dy.cuda())
        assert y.dtype == d.dtype == DT[dt] and y.shape == (n, width) and d.shape == (vocab, width)
        _check(table, tokens, dy, scale, y, d)
        plain = F.embedding(w.detach(), tokens.cuda(), scale=scale)
        assert not plain.requires_grad and torch.equal(plain.nan_to_num(5), y.detach().nan_to_num(5))


def test_values_without_scale_are_the_tables():
    F = _F()
    table = _normal((50, 40), torch.bfloat16, 3)
    table[3, 4], table[5, 6] = float("inf"), -0.0
    t = torch.arange(50)
    y = F.embedding(table.cuda(), t.cuda())
    assert torch.equal(y.cpu().view(torch.int16), table.view(torch.int16))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layouts(dt):
    """Tokens of any shape, int32, strided; a table and cotangents that are slices, broadcast or transposed."""
    F = _F()
    wide = _normal((300, 101), DT[dt], 4)
    table = wide[:, 3:80]
    tokens = _tokens("none", 60, 300).clamp(min=-1, max=300).reshape(3, 20)
    dev = wide.cuda()[:, 3:80].requires_grad_(True)
    for tok in (tokens.cuda(), tokens.to(torch.int32).cuda(), tokens.t().contiguous().cuda().t()):
        y = F.embedding(dev, tok, 0.5)
        for dy in (_normal((3, 20, 77), DT[dt], 5), _normal((3, 1, 77), DT[dt], 6).expand(3, 20, 77),
                   _normal((77, 20, 3), DT[dt], 6).permute(2, 1, 0), torch.ones((), dtype=DT[dt]).expand(3, 20, 77),
                   _normal((3, 20, 100), DT[dt], 8)[..., 11:88]):
            d, = torch.autograd.grad(y, dev, dy.cuda(), retain_graph=True)
            _check(table, tokens, dy, 0.5, y, d)
    back = _normal((77, 300), DT[dt], 9)
    y = F.embedding(back.cuda().t(), tokens.cuda())
    _check(back.t(), tokens, torch.zeros(3, 20, 77), 1.0, y, None)
    one = F.embedding(dev, torch.tensor(7, device="cuda"))
    assert one.shape == (77,) and torch.equal(one.detach().cpu(), table[7])


def test_empty():
    F = _F()
    w = _normal((9, 20), torch.float32, 1).cuda().requires_grad_(True)
    y = F.embedding(w, torch.zeros((0, 4), dtype=torch.int64, device="cuda"))
    assert y.shape == (0, 4, 20)
    d, = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert d.shape == w.shape and not bool(d.any())
    none = torch.zeros((9, 0), device="cuda", requires_grad=True)
    y = F.embedding(none, torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert y.shape == (3, 0) and torch.autograd.grad(y.sum(), none)[0].shape == (9, 0)


def test_same_bits_and_streams():
    """Two calls give the same bits, also on another stream and from a captured graph's replays."""
    F = _F()
    table = _normal((2000, 300), torch.bfloat16, 1).cuda().requires_grad_(True)
    tokens = _tokens("runs", 3000, 50).cuda()
    dy = _normal((3000, 300), torch.bfloat16, 2).cuda()

    def work():
        y = F.embedding(table, tokens, 3.0)
        return (y,) + torch.autograd.grad(y, table, dy)
    want = [t.detach().clone() for t in work()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(work(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for rep in range(3):
        tokens.copy_(_tokens("runs", 3000, 50 + 700 * rep, seed=rep))
        dy.copy_(_normal((3000, 300), torch.bfloat16, 20 + rep))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, work())), rep


def test_bounds():
    """Nothing but the outputs and the workspace is written."""
    from tests.test_gpu_row_ops_bounds import Guarded, _lib, _ptr, _stream
    L, lib = _lib()
    for dtype, code in ((torch.bfloat16, 1), (torch.float32, 0)):
        for n, vocab, width in ((1, 1, 1), (200, 5, 13), (1000, 700, 1025), (70, 66000, 3)):
            e = dtype.itemsize
            table, dy, tokens = _normal((vocab, width), dtype, 1), _normal((n, width), dtype, 2), _tokens("none", n, vocab)
            y, d = Guarded(n * width, dtype, e), Guarded(vocab * width, dtype, e)
            need = lib.pratchya_embedding_bwd_workspace_bytes(n, vocab, width)
            ws = Guarded(need, torch.uint8)
            dev = [t.cuda() for t in (table, dy, tokens)]
            assert lib.pratchya_embedding(_ptr(dev[0]), width, code, _ptr(dev[2]), n, vocab, width, 2.0, y.p,
                                          _stream()) == L.OK
            assert lib.pratchya_embedding_bwd(_ptr(dev[1]), width, code, _ptr(dev[2]), n, vocab, width, 2.0, d.p, ws.p,
                                              need, _stream()) == L.OK
            torch.cuda.synchronize()
            assert y.untouched() and d.untouched() and ws.untouched()
            _check(table, tokens, dy, 2.0, y.t.reshape(n, width), d.t.reshape(vocab, width))


def test_refusals():
    F = _F()
    w = torch.zeros((4, 8), device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad, error in ((lambda: F.embedding(w.half(), t), TypeError), (lambda: F.embedding(w, t.float()), TypeError),
                       (lambda: F.embedding(w[0], t), ValueError), (lambda: F.embedding(w[:0], t), ValueError),
                       (lambda: F.embedding(w, t.cpu()), RuntimeError), (lambda: F.embedding(w, [1, 2]), TypeError)):
        with pytest.raises(error):
            bad()
    y = F.embedding(w.requires_grad_(True), t)
    d, = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        d.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        F.embedding(fwd.make_dual(w.detach(), torch.ones_like(w)), t)
