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
    assert bwd(vocab=1 << 27) == L.EUNSUPPORTED and bwd(n=100, width=1 << 25) == L.EUNSUPPORTED
    need = lib.pratchya_embedding_bwd_workspace_bytes
    assert need(0, 1, 8) > 0 and need(1000, 50, 64) >= 8 * 1000 + 4 * 51 and need(1 << 31, 5, 8) == 0
