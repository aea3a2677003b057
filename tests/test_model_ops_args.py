"""Argument checks of the C entry points at a model's ends and in its time mixing
(embedding, linear attention, cross entropy of a head): they return before any launch,
without a GPU."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(1 << 20)          # aligned, never dereferenced


def _L():
    from pratchya_amd import _lib
    return _lib, _lib.load()


def test_embedding():
    L, lib = _L()

    def fwd(table=FAKE, ld=8, dtype=1, tokens=FAKE, n=4, vocab=9, width=8, y=FAKE):
        return lib.pratchya_embedding(table, ld, dtype, tokens, n, vocab, width, 1.0, y, None)
    assert fwd(n=0) == L.OK and fwd(width=0) == L.OK
    for bad in (dict(dtype=2), dict(n=-1), dict(vocab=0), dict(width=-1), dict(ld=-8), dict(table=None),
                dict(tokens=None), dict(y=None)):
        assert fwd(**bad) == L.EINVAL, bad
        assert b"embedding" in lib.pratchya_last_error()
    assert fwd(n=1 << 31) == L.EUNSUPPORTED and fwd(vocab=1 << 31) == L.EUNSUPPORTED
    assert fwd(n=1 << 27) == L.EUNSUPPORTED and fwd(n=1 << 24, width=1 << 16) == L.EUNSUPPORTED

    def bwd(dy=FAKE, dtype=1, tokens=FAKE, n=4, vocab=9, width=8, d=FAKE, ws=FAKE, ws_bytes=1 << 60):
        return lib.pratchya_embedding_bwd(dy, width, dtype, tokens, n, vocab, width, 1.0, d, ws, ws_bytes, None)
    assert bwd(width=0) == L.OK
    for bad in (dict(dtype=2), dict(n=-1), dict(vocab=0), dict(dy=None), dict(tokens=None), dict(d=None), dict(ws=None),
                dict(ws_bytes=8), dict(ws=ctypes.c_void_p((1 << 20) + 8))):
        assert bwd(**bad) == L.EINVAL, bad
        assert b"embedding_bwd" in lib.pratchya_last_error()
    assert bwd(vocab=1 << 30, width=1 << 10) == L.EUNSUPPORTED and bwd(n=1 << 27) == L.EUNSUPPORTED and bwd(n=100, width=1 << 25) == L.EUNSUPPORTED
    need = lib.pratchya_embedding_bwd_workspace_bytes
    assert need(0, 1, 8) > 0 and need(1000, 50, 64) >= 8 * 1000 + 4 * 51 and need(1 << 31, 5, 8) == 0


def test_linear_cross_entropy():
    L, lib = _L()

    def fwd(x=FAKE, ldx=64, w=FAKE, ldw=128, dtype=1, rows=0, t=FAKE, n=64, C=64, V=128, a=0.0, loss=FAKE, ws=FAKE,
            ws_bytes=1 << 60):
        return lib.pratchya_linear_cross_entropy(x, ldx, w, ldw, dtype, rows, t, n, C, V, a, loss, None, ws, ws_bytes, None)
    assert fwd(n=0) == L.OK
    for bad in (dict(dtype=2), dict(n=-1), dict(C=0), dict(V=0), dict(ldx=-1), dict(a=-0.5), dict(a=1.5),
                dict(a=float("nan")), dict(x=None), dict(w=None), dict(t=None), dict(loss=None), dict(ws=None),
                dict(ws_bytes=8), dict(ws=ctypes.c_void_p((1 << 20) + 16))):
        assert fwd(**bad) == L.EINVAL, bad
        assert b"linear_cross_entropy" in lib.pratchya_last_error()
    for big in (dict(n=1 << 24), dict(n=1 << 20, C=4096), dict(V=1 << 31), dict(C=1 << 31), dict(n=1 << 21, dtype=0)):
        assert fwd(**big) == L.EUNSUPPORTED, big

    def bwd(x=FAKE, w=FAKE, dtype=1, t=FAKE, stats=FAKE, g=FAKE, n=64, C=64, V=128, a=0.0, dx=FAKE, dw=FAKE, ws=FAKE,
            ws_bytes=1 << 60):
        return lib.pratchya_linear_cross_entropy_bwd(x, C, w, V, dtype, 0, t, stats, g, n, C, V, a, dx, dw, ws, ws_bytes,
                                                     None)
    assert bwd(dx=None, dw=None) == L.OK and bwd(n=0, dw=None) == L.OK
    for bad in (dict(dtype=2), dict(a=2.0), dict(x=None), dict(t=None), dict(stats=None), dict(g=None), dict(ws=None),
                dict(ws_bytes=64)):
        assert bwd(**bad) == L.EINVAL, bad
        assert b"linear_cross_entropy_bwd" in lib.pratchya_last_error()
    need = lib.pratchya_linear_cross_entropy_workspace_bytes
    # a large vocabulary's logits are never whole
    assert 0 < need(FAKE, 4096, FAKE, 65536, 1, 0, 8192, 4096, 65536, 0, 0) < 1 << 29
    assert need(FAKE, 4096, FAKE, 65536, 1, 0, 8192, 4096, 65536, 1, 1) < 3 << 29


def test_names_without_gpu():
    """Arguments that a user can get wrong are refused before the library is asked."""
    import torch
    from pratchya_amd import functional as F
    x, t = torch.zeros((2, 8)), torch.zeros(2).long()
    for call in (lambda: F.embedding(x, t), lambda: F.linear_cross_entropy(x, x.t(), t)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_linear_attention():
    L, lib = _L()
    st = (ctypes.c_int64 * 15)(*[8] * 15)

    def fwd(q=FAKE, dtype=1, g=FAKE, gdt=0, st=st, B=2, T=5, H=3, dk=8, dv=8, out=FAKE, s=FAKE, starts=None):
        return lib.pratchya_linear_attention(q, q, q, dtype, g, gdt, st, None, None, B, T, H, dk, dv, 1.0, 1, out, s, starts,
                                             None)
    assert fwd(B=0) == L.OK
    for bad in (dict(dtype=2), dict(gdt=2), dict(B=-1), dict(T=-1), dict(H=0), dict(dk=0), dict(dv=0), dict(q=None),
                dict(g=None), dict(st=None), dict(out=None), dict(s=None), dict(T=4096)):
        assert fwd(**bad) == L.EINVAL, bad
        assert b"linear_attention" in lib.pratchya_last_error()
    for big in (dict(dk=129), dict(dv=129), dict(T=1 << 31), dict(B=1 << 24), dict(B=1 << 25, H=1)):
        assert fwd(**big) == L.EUNSUPPORTED, big
    assert lib.pratchya_linear_attention_starts_floats(1, 200, 1, 8, 8, 1, 1) == 0
    assert lib.pratchya_linear_attention_starts_floats(1, 4096, 1, 8, 8, 1, 1) > 0

    def bwd(q=FAKE, dtype=1, T=5, dk=8, dq=FAKE, dg=FAKE, s=FAKE, ds=FAKE, starts=None, ws=FAKE, ws_bytes=1 << 60):
        return lib.pratchya_linear_attention_bwd(q, q, q, dtype, FAKE, 0, st, None, None, s, starts, FAKE, ds, 2, T, 3, dk,
                                                 8, 1.0, dq, FAKE, FAKE, dg, None, ws, ws_bytes, None)
    for bad in (dict(dtype=2), dict(dk=0), dict(q=None), dict(dq=None), dict(s=None), dict(T=4096), dict(ws=None),
                dict(ws_bytes=8)):
        assert bwd(**bad) == L.EINVAL, bad
        assert b"linear_attention_bwd" in lib.pratchya_last_error()
    assert bwd(dk=129) == L.EUNSUPPORTED

    def step(q=FAKE, dtype=1, B=2, H=3, dk=8, s=FAKE, out=FAKE):
        return lib.pratchya_linear_attention_step(q, q, q, dtype, FAKE, 0, st, s, B, H, dk, 8, 1.0, out, None)
    assert step(B=0) == L.OK
    for bad in (dict(dtype=3), dict(B=-1), dict(H=0), dict(dk=0), dict(q=None), dict(s=None), dict(out=None),
                dict(s=ctypes.c_void_p((1 << 20) + 4))):
        assert step(**bad) == L.EINVAL, bad
        assert b"linear_attention_step" in lib.pratchya_last_error()
    assert step(dk=200) == L.EUNSUPPORTED
