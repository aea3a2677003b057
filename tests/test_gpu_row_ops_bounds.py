"""What the row operators' kernels write, and nothing else: outputs and workspaces lie
inside larger buffers of a known value through the C entry points, and what is around
them keeps it.  A bad value of a norm reaches its own columns' weight gradient only."""
import ctypes
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
PAD = 4096
MARK = 0xA5


class Guarded:
    """n elements of dtype at `shift` bytes past an aligned address, between PAD bytes on either side."""
    def __init__(self, n, dtype, shift=0):
        self.size = n * dtype.itemsize
        self.buf = torch.full((self.size + 2 * PAD + shift,), MARK, dtype=torch.uint8, device="cuda")
        self.at = PAD + shift
        self.t = self.buf[self.at:self.at + self.size].view(dtype)
        self.p = ctypes.c_void_p(self.buf.data_ptr() + self.at)

    def untouched(self):
        b = self.buf
        return bool((b[:self.at] == MARK).all()) and bool((b[self.at + self.size:] == MARK).all())


def _lib():
    from pratchya_amd import _lib
    return _lib, _lib.load()


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,groups,blk", [
    (1, 1, 1, 0), (1, 3, 1, 0), (5, 7, 1, 0), (1, 9, 1, 0), (4, 13, 1, 0), (3, 65, 1, 0), (6, 30, 6, 0), (1, 30, 2, 0),
    (1, 1027, 1, 0), (7, 1029, 3, 0), (2, 4097, 1, 0), (1, 6151, 1, 0), (700, 1030, 1, 0), (1, 16391, 1, 0),
    (3, 16384, 1, 0), (2, 33001, 1, 0), (1, 16, 1, 16), (3, 1024, 1, 128), (5, 192, 1, 32), (40, 256, 1, 64),
    (1, 12288, 1, 64), (9, 4160, 1, 0)])
def test_layer_norm(rows, width, groups, blk, dt):
    L, lib = _lib()
    gen = torch.Generator().manual_seed(rows + width)
    x, dy = (torch.randn((rows, width), generator=gen).to(DT[dt]).cuda() for _ in range(2))
    w, b = (torch.randn(width, generator=gen).cuda() for _ in range(2))
    code = 1 if dt == "bf16" else 0
    e = DT[dt].itemsize
    y, stats = Guarded(rows * width, DT[dt], e), Guarded(rows * groups * 2, torch.float32)
    x8, sc8, sc32 = ((Guarded(rows * width, torch.uint8), Guarded(rows * width // blk, torch.uint8),
                      Guarded(rows * width // (blk * (blk // 16)), torch.float32)) if blk else (None,) * 3)
    held = [g for g in (y, stats, x8, sc8, sc32) if g]
    p8 = [g.p if g else None for g in (x8, sc8, sc32)]
    if blk:
        assert lib.pratchya_layer_norm_stores(width, groups, blk)
    assert lib.pratchya_layer_norm(_ptr(x), width, code, _ptr(w), 0, _ptr(b), 0, rows, width, groups, EPS, y.p, stats.p,
                                   *p8, blk, _stream()) == L.OK
    dx, dw, db = Guarded(rows * width, DT[dt], e), Guarded(width, torch.float32, 4), Guarded(width, torch.bfloat16, 2)
    need = lib.pratchya_layer_norm_bwd_workspace_bytes(rows, width, groups)
    ws = Guarded(need // 4, torch.float32)
    src = (x8.p, 0, 2, sc8.p, sc32.p, blk) if blk else (_ptr(x), width, code, None, None, 0)
    assert lib.pratchya_layer_norm_bwd(*src, _ptr(dy), width, code, _ptr(w), 0, stats.p, rows, width, groups, dx.p, dw.p,
                                       0, db.p, 1, ws.p, need, _stream()) == L.OK
    torch.cuda.synchronize()
    for g in held + [dx, dw, db, ws]:
        assert g.untouched()
    want, bound = R.layer_norm(x.cpu(), w.cpu(), b.cpu(), EPS, groups, dy.cpu(), blk)
    for g, v, lim, n in zip((y, dx, dw, db), want, bound, ("y", "dx", "dw", "db")):
        R.close(g.t, v, lim, n)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,blk", [(1, 1, 0), (3, 7, 0), (1, 4095, 0), (33, 1023, 0), (2, 16, 16), (5, 2176, 128),
                                            (7, 96, 32), (3, 320, 64)])
def test_activation(rows, width, blk, dt):
    L, lib = _lib()
    gen = torch.Generator().manual_seed(rows + width)
    wide = torch.randn((rows, width + 5), generator=gen).to(DT[dt]).cuda()
    code, e = (1 if dt == "bf16" else 0), DT[dt].itemsize
    for x, ld in ((wide[:, 2:2 + width], width + 5), (wide[:, 2:2 + width].contiguous(), width)):
        n = rows * width
        k = 1 if not blk else math.gcd(max(1, blk // 16), n // blk)
        y, dx = Guarded(n, DT[dt], e), Guarded(n, DT[dt], e)
        x8, sc8, sc32 = ((Guarded(n, torch.uint8), Guarded(n // blk, torch.uint8), Guarded(n // blk // k, torch.float32))
                         if blk else (None,) * 3)
        p8 = [g.p if g else None for g in (x8, sc8, sc32)]
        assert lib.pratchya_activation(_ptr(x), ld, code, 1, rows, width, y.p, *p8, blk, _stream()) == L.OK
        src = (x8.p, 0, 2, sc8.p, sc32.p, blk) if blk else (_ptr(x), ld, code, None, None, 0)
        assert lib.pratchya_activation_bwd(*src, _ptr(x), ld, code, 1, rows, width, dx.p, _stream()) == L.OK
        torch.cuda.synchronize()
        for g in (y, dx, x8, sc8, sc32):
            assert g is None or g.untouched()
        want, bound = R.activation(x.cpu(), "silu", x.cpu(), blk)
        R.close(y.t, want[0], bound[0], "y")
        R.close(dx.t, want[1], bound[1], "dx")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 0), (5, 100, 20), (2, 4099, 5), (1, 20001, 64), (3, 2049, 0),
                                            (520, 2051, 0), (4, 1023, 33), (2, 70001, 1)])
def test_token_logprobs(rows, vocab, top, dt):
    L, lib = _lib()
    gen = torch.Generator().manual_seed(rows + vocab)
    x = torch.randn((rows, vocab), generator=gen).to(DT[dt]).cuda()
    tokens = torch.randint(0, vocab, (rows,), generator=gen).cuda()
    code, e = (1 if dt == "bf16" else 0), DT[dt].itemsize
    lp, h, st = Guarded(rows, torch.float32), Guarded(rows, torch.float32, 4), Guarded(3 * rows, torch.float32)
    need = lib.pratchya_token_logprobs_workspace_bytes(rows, vocab, top) if top else 0
    best, at = (Guarded(rows * top, torch.float32), Guarded(rows * top, torch.int64)) if top else (None, None)
    ws = Guarded(need, torch.uint8) if need else None
    assert lib.pratchya_token_logprobs(_ptr(x), vocab, code, _ptr(tokens), rows, vocab, top, lp.p, h.p, st.p,
                                       best.p if top else None, at.p if top else None, ws.p if ws else None, need,
                                       _stream()) == L.OK
    g = torch.randn(rows, generator=gen).cuda()
    dx = Guarded(rows * vocab, DT[dt], e)
    assert lib.pratchya_token_logprobs_bwd(_ptr(x), vocab, code, _ptr(tokens), st.p, _ptr(g), _ptr(g), rows, vocab, dx.p,
                                           _stream()) == L.OK
    torch.cuda.synchronize()
    for b in (lp, h, st, best, at, ws, dx):
        assert b is None or b.untouched()
    want, bound = R.token_logprobs(x.cpu(), tokens.cpu(), g.cpu(), g.cpu())
    for b, v, lim in zip((lp, h, dx), want, bound):
        R.close(b.t, v, lim, "result")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,groups", [(12, 256, 4), (12, 4096, 1), (12, 1000, 1), (600, 520, 1), (9, 17000, 1)])
def test_weight_gradient_beside_bad_segments(rows, width, groups, dt):
    """An infinity and a NaN: dw is NaN in their segments' columns and within its bound in all others."""
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(rows + width)
    x, dy = (torch.randn((rows, width), generator=gen).to(DT[dt]) for _ in range(2))
    w, b = (torch.randn(width, generator=gen) for _ in range(2))
    D = width // groups
    bad = x.clone()
    bad[3, 1], bad[7, min(2 * D, width) - 1] = float("inf"), float("nan")
    args = [t.cuda().requires_grad_(True) for t in (bad, w, b)]
    y = F.layer_norm(*args, groups=groups)
    dx, dw, db = torch.autograd.grad(y, args, dy.cuda())
    want, bound = R.layer_norm(x, w, b, EPS, groups, dy)
    spoilt = torch.zeros(width, dtype=torch.bool)
    spoilt[:min(2 * D, width)] = True
    assert torch.equal(torch.isnan(dw.cpu()), spoilt)
    if not bool(spoilt.all()):
        R.close(dw[~spoilt.cuda()], want[2][~spoilt], bound[2][~spoilt], "dw")
    R.close(db, want[3], bound[3], "db")
    keep = [r for r in range(rows) if r not in (3, 7)]
    R.close(dx[keep], want[1][keep], bound[1][keep], "dx")
