"""Workspace sizes of the head's cross entropy and of linear attention over the range of their
arguments, without a GPU: no overflow, no size of nothing, refusals instead."""
import itertools

import pytest

FAKE = 1 << 20


def _lib():
    from pratchya_amd import _lib
    return _lib, _lib.load()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows", [0, 1])
def test_cross_entropy(rows, dtype):
    _, lib = _lib()
    for n, C, V in itertools.product((1, 255, 256, 1000, 65536, 1 << 23), (1, 256, 257, 4096, 1 << 20),
                                     (1, 256, 257, 50021, 262144, 0x7FFFFF00)):
        size = lib.pratchya_linear_cross_entropy_workspace_bytes
        sizes = [size(FAKE, C, FAKE, C if rows else V, dtype, rows, n, C, V, dx, dw) for dx, dw in ((0, 0), (1, 0), (0, 1), (1, 1))]
        if any(sizes):
            # at least the rows' planes; the loss alone, unlike the gradients, keeps the rows' statistics
            assert all(s >= (2 if dtype else 6) * n * C for s in sizes), (n, C, V)
            assert sizes[3] >= max(sizes[1:3])
        else:
            assert b"linear_cross_entropy" in lib.pratchya_last_error()
            assert n * C * (2 if dtype else 6) > 1 << 20


@pytest.mark.parametrize("dtype", [0, 1])
def test_pieces_are_bounded(dtype):
    """What is held besides operands: a piece of the gradients, 5% of what bf16 logits take."""
    _, lib = _lib()
    for n, C, V in ((8192, 4096, 65536), (4096, 2048, 131072), (512, 1024, 262144), (100, 64, 1 << 20)):
        size = lib.pratchya_linear_cross_entropy_workspace_bytes
        assert size(FAKE, C, FAKE, V, dtype, 0, n, C, V, 0, 0) < 0.1 * n * V + 14 * n * C + (1100 << 20)
        assert size(FAKE, C, FAKE, V, dtype, 0, n, C, V, 1, 1) < 30 * n * C + (2200 << 20)


def test_linear_attention():
    L, lib = _lib()
    for B, T, H, d, dtype, train in itertools.product((1, 5, 1 << 20), (1, 63, 1000, 8192, 0x7FFFFF00), (1, 100), (1, 64, 128),
                                                      (0, 1), (0, 1)):
        floats = lib.pratchya_linear_attention_starts_floats(B, T, H, d, d, dtype, train)
        assert floats >= 0 and (floats == 0 or floats >= 2 * B * H * d * d)
        ws = lib.pratchya_linear_attention_bwd_workspace_bytes(B, T, H, d, d, dtype)
        assert ws == 0 or ws >= 4 * B * H * T
    assert lib.pratchya_linear_attention_starts_floats(1, 255, 1, 64, 64, 1, 1) == 0
    assert lib.pratchya_linear_attention_starts_floats(1, 512, 1, 64, 64, 1, 1) > 0
