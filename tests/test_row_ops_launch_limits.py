"""Calls of the row operators' C entry points that no single launch can hold (2^32
threads along x, 65535 workgroups along y) are refused before any launch, so this runs
without a GPU; no buffer is read or written."""
import ctypes

import pytest
import torch

# a call that were not refused would launch on addresses that do not exist
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="runs where nothing can be launched")

FAKE = ctypes.c_void_p(1 << 20)          # aligned, never dereferenced
BIG = 1 << 60


def _L():
    from pratchya_amd import _lib
    return _lib, _lib.load()


def _refused(L, lib, rc, what):
    assert rc == L.EUNSUPPORTED, (what, rc, lib.pratchya_last_error())
    assert what.encode() in lib.pratchya_last_error()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,vocab,top", [((1 << 26) - 3, 16, 0), (1 << 24, 2049, 0), ((1 << 24) + 5, 70000, 0),
                                            (1 << 24, 16, 1), (1 << 23, 5000, 3), (1 << 18, 1 << 20, 64)])
def test_token_logprobs(rows, vocab, top, dtype):
    L, lib = _L()
    best = FAKE if top else None
    _refused(L, lib, lib.pratchya_token_logprobs(FAKE, vocab, dtype, FAKE, rows, vocab, top, FAKE, FAKE, FAKE, best, best,
                                                 FAKE, BIG, None), "token_logprobs")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,vocab", [((1 << 26) + 1, 16), (1 << 24, 3000), (1 << 20, 65536)])
def test_token_logprobs_bwd(rows, vocab, dtype):
    L, lib = _L()
    _refused(L, lib, lib.pratchya_token_logprobs_bwd(FAKE, vocab, dtype, FAKE, FAKE, FAKE, None, rows, vocab, FAKE, None),
             "token_logprobs_bwd")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,width,ld", [(1 << 20, 1 << 16, 1 << 16), (1 << 20, 1 << 16, 1 << 17),
                                           ((1 << 31) - 1, 256, 256)])
def test_activation(rows, width, ld, dtype):
    L, lib = _L()
    _refused(L, lib, lib.pratchya_activation(FAKE, ld, dtype, 1, rows, width, FAKE, None, None, None, 0, None),
             "activation")
    _refused(L, lib, lib.pratchya_activation_bwd(FAKE, ld, dtype, None, None, 0, FAKE, ld, dtype, 1, rows, width, FAKE,
                                                 None), "activation_bwd")
    if ld == width:
        _refused(L, lib, lib.pratchya_activation_bwd(FAKE, ld, 2, FAKE, FAKE, 32, FAKE, ld, dtype, 1, rows, width, FAKE,
                                                     None), "activation_bwd")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,width,groups", [(1 << 22, 16385, 1), (1 << 11, 1 << 26, 1 << 11),
                                               (1, 1 << 30, 1 << 20), (1, 1 << 31, 1 << 20)])
def test_layer_norm(rows, width, groups, dtype):
    L, lib = _L()
    _refused(L, lib, lib.pratchya_layer_norm(FAKE, width, dtype, None, 0, None, 0, rows, width, groups, 1e-5, FAKE, FAKE,
                                             None, None, None, 0, None), "layer_norm")
    _refused(L, lib, lib.pratchya_layer_norm_bwd(FAKE, width, dtype, None, None, 0, FAKE, width, dtype, None, 0, FAKE,
                                                 rows, width, groups, FAKE, FAKE, 0, FAKE, 0, FAKE, BIG, None),
             "layer_norm_bwd")


@pytest.mark.parametrize("rows,width,groups", [(2, 1 << 28, 1), (1, 1 << 29, 2)])
def test_layer_norm_columns(rows, width, groups):
    """The parameters' gradients are joined by a launch of 16 threads a column."""
    L, lib = _L()
    _refused(L, lib, lib.pratchya_layer_norm_bwd(FAKE, width, 1, None, None, 0, FAKE, width, 1, None, 0, FAKE, rows, width,
                                                 groups, FAKE, FAKE, 0, None, 0, FAKE, BIG, None), "layer_norm_bwd")
