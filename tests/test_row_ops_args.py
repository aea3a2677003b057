"""Argument checks of the row operators' C entry points (layer norm, activations,
token log probabilities): they return before any launch, without a GPU."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(1 << 20)          # aligned, never dereferenced


def _L():
    from pratchya_amd import _lib
    return _lib


def _ln(lib, x=FAKE, dtype=1, w=FAKE, w_dtype=0, rows=4, width=96, groups=1, y=FAKE, x8=None, blk=0):
    return lib.pratchya_layer_norm(x, width, dtype, w, w_dtype, None, 0, rows, width, groups, 1e-5, y, None, x8, x8, x8,
                                   blk, None)


def test_layer_norm():
    L = _L()
    lib = L.load()
    assert _ln(lib, rows=0) == L.OK and _ln(lib, width=0) == L.OK
    for bad in (dict(groups=5), dict(groups=0), dict(rows=-1), dict(dtype=2), dict(w_dtype=7), dict(x=None),
                dict(y=None)):
        assert _ln(lib, **bad) == L.EINVAL, bad
        assert b"layer_norm" in lib.pratchya_last_error()
    assert _ln(lib, rows=1 << 40) == L.EUNSUPPORTED
    assert lib.pratchya_layer_norm_stores(2176, 1, 128) == 0       # groups of 8 blocks over 17 blocks a row
    assert lib.pratchya_layer_norm_stores(1024, 1, 24) == 0
    assert _ln(lib, width=2176, x8=FAKE, blk=128) == L.EUNSUPPORTED


def _lnb(lib, x=FAKE, x_dtype=1, sc=None, blk=0, dy=FAKE, dtype=1, stats=FAKE, rows=4, width=96, groups=1, ws=FAKE,
         ws_bytes=1 << 30):
    return lib.pratchya_layer_norm_bwd(x, width, x_dtype, sc, sc, blk, dy, width, dtype, None, 0, stats, rows, width,
                                       groups, FAKE, FAKE, 0, FAKE, 0, ws, ws_bytes, None)


def test_layer_norm_bwd():
    L = _L()
    lib = L.load()
    assert _lnb(lib, rows=0) == L.OK
    for bad in (dict(groups=5), dict(dtype=2), dict(x_dtype=0), dict(x=None), dict(dy=None), dict(stats=None),
                dict(ws=None), dict(ws_bytes=8), dict(ws=ctypes.c_void_p((1 << 20) + 2)), dict(x_dtype=2, blk=32),
                dict(x_dtype=2, blk=36, sc=FAKE), dict(x_dtype=2, blk=0, sc=FAKE)):
        assert _lnb(lib, **bad) == L.EINVAL, bad
        assert b"layer_norm_bwd" in lib.pratchya_last_error()
    for rows in (1, 7, 1000, 100000):
        assert lib.pratchya_layer_norm_bwd_workspace_bytes(rows, 4096, 1) >= 2 * 4096 * 4


def test_activation():
    L = _L()
    lib = L.load()

    def fwd(x=FAKE, dtype=1, kind=0, rows=4, width=96, y=FAKE, x8=None, sc=FAKE, blk=0):
        return lib.pratchya_activation(x, width, dtype, kind, rows, width, y, x8, sc, sc, blk, None)

    def bwd(x=FAKE, x_dtype=1, sc=None, blk=0, dy=FAKE, dtype=1, kind=0, rows=4, width=96):
        return lib.pratchya_activation_bwd(x, width, x_dtype, sc, sc, blk, dy, width, dtype, kind, rows, width, FAKE,
                                           None)
    assert fwd(rows=0) == L.OK and bwd(width=0) == L.OK
    for bad in (dict(kind=3), dict(kind=-1), dict(dtype=2), dict(rows=-1), dict(x=None), dict(y=None)):
        assert fwd(**bad) == L.EINVAL, bad
    for bad in (dict(kind=3), dict(dtype=2), dict(x_dtype=0), dict(x=None), dict(dy=None), dict(x_dtype=2, blk=32),
                dict(x_dtype=2, blk=36, sc=FAKE), dict(x_dtype=2, sc=FAKE)):
        assert bwd(**bad) == L.EINVAL, bad
        assert b"activation_bwd" in lib.pratchya_last_error()


def test_token_logprobs():
    L = _L()
    lib = L.load()

    def fwd(x=FAKE, dtype=1, tokens=FAKE, rows=4, vocab=96, top=0, out=FAKE, best=None):
        return lib.pratchya_token_logprobs(x, vocab, dtype, tokens, rows, vocab, top, out, None, None, best, best, None,
                                           0, None)
    assert fwd(rows=0) == L.OK
    for bad in (dict(dtype=2), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(top=-1), dict(top=65),
                dict(top=97, vocab=96), dict(top=3), dict(x=None), dict(tokens=None), dict(out=None)):
        assert fwd(**bad) == L.EINVAL, bad
        assert b"token_logprobs" in lib.pratchya_last_error()
    assert fwd(rows=1 << 31) == L.EUNSUPPORTED
    assert lib.pratchya_token_logprobs_workspace_bytes(4, 96, 20) == 0 and fwd(vocab=1 << 20, top=3, best=FAKE) == L.EINVAL
    assert b"workspace" in lib.pratchya_last_error()

    def bwd(x=FAKE, dtype=1, stats=FAKE, rows=4, vocab=96, dx=FAKE):
        return lib.pratchya_token_logprobs_bwd(x, vocab, dtype, FAKE, stats, None, None, rows, vocab, dx, None)
    assert bwd(rows=0) == L.OK
    for bad in (dict(dtype=2), dict(vocab=0), dict(x=None), dict(stats=None), dict(dx=None)):
        assert bwd(**bad) == L.EINVAL, bad
    assert bwd(rows=1 << 31) == L.EUNSUPPORTED


def test_names_without_gpu():
    """Arguments that a user can get wrong are refused before the library is asked."""
    import torch
    from pratchya_amd import functional as F
    x = torch.zeros((2, 8))
    for call in (lambda: F.layer_norm(x), lambda: F.activation(x), lambda: F.token_logprobs(x, torch.zeros(2).long())):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
