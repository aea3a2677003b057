"""What linear_cross_entropy asks of memory below 256 rows, by the library's size query: pieces of
planes and sums, no f32 copy of the weight's gradient."""
import pytest

FAKE = 1 << 20
MB = 1 << 20


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("n,C,V", [(128, 4096, 65536), (255, 8192, 128256), (64, 4096, 262144), (1, 2048, 50257), (40, 4100, 20003)])
def test_few_rows(n, C, V, rows, dtype):
    from pratchya_amd import _lib
    size = _lib.load().pratchya_linear_cross_entropy_workspace_bytes
    n64, planes = (n + 63) // 64 * 64, 2 if dtype else 6
    for back in ((0, 0), (1, 0), (0, 1), (1, 1)):
        got = size(FAKE, C, FAKE, C if rows else V, dtype, rows, n, C, V, *back)
        # logits and their gradient, x's planes, partial sums of x's gradient, what products hold of slices
        bound = (4 + planes) * n64 * (V + 64) + planes * n64 * (C + 64) + 140 * n * (C + 64) + 64 * MB
        if not (dtype == 1 and C % 64 == 0 and V % 64 == 0):
            bound += 512 * MB      # a piece of the weight's planes
        plain = C % 8 == 0 and V % 8 == 0
        if back[1]:
            bound += (32 if plain else 256) * MB
        assert 0 < got < bound, (back, got / MB, bound / MB)
    if (n, dtype) == (128, 1):
        assert size(FAKE, C, FAKE, C if rows else V, 1, rows, n, C, V, 1, 1) < 150 * MB


@pytest.mark.parametrize("rows", [0, 1])
def test_weights_inside_wider_arrays(rows):
    """A table of rows far apart, or [C, V] columns of a wide array: pieces that the products take."""
    from pratchya_amd import _lib
    lib = _lib.load()
    size = lib.pratchya_linear_cross_entropy_workspace_bytes
    for n, C, V, ld in ((64, 4096, 262144, 8192), (64, 64, 20032, 131072), (1, 4096, 65536, 1 << 16), (200, 2048, 128256, 40000),
                        (300, 256, 40000, 100000), (64, 64, 1024, 30000000), (255, 192, 100096, 200000)):
        if not rows and ld < V:
            continue
        for back in ((0, 0), (1, 0), (0, 1), (1, 1)):
            got = size(FAKE, C, FAKE, ld, 1, rows, n, C, V, *back)
            # at most as a copy of the weight's pieces would need
            assert 0 < got < size(FAKE, C, FAKE, ld + 1, 1, rows, n, C, V, *back) + 4 * n * V, (n, C, V, ld, back)


def _by_tiles(n, C, V, ldx, ldw, rows):
    """Whether the loss takes each row's statistics from the products' tiles, of 128 columns each and
    12 bytes, with no logits written: what it holds for 2 n rows more than for n."""
    from pratchya_amd import _lib
    size = _lib.load().pratchya_linear_cross_entropy_workspace_bytes
    one, two = (size(FAKE, ldx, FAKE, ldw, 1, rows, m, C, V, 0, 0) for m in (n, 2 * n))
    assert 0 < one and 0 < two
    more, statistics = two - one - 2 * n * C, 12 * n * (V // 128)      # but for x's planes
    return 0.4 * statistics < more < 1.6 * statistics      # the vocabulary's end may go by written logits, in one or both


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("C,V", [(4096, 65536), (8192, 131072), (8192, 152064), (4096, 262144 + 4096)])
def test_large_heads_keep_no_logits(C, V, rows):
    """Also where the weight's size exceeds 31 bits."""
    assert _by_tiles(8192, C, V, C, C if rows else V, rows)


def test_rows_far_apart_keep_no_logits():
    """Rows of x and of a table that lie beyond 31 bits in place."""
    assert _by_tiles(8192, 4096, 65536, 1 << 18, 4096, 1)
    assert _by_tiles(8192, 4096, 65536, 4096, 1 << 19, 1)
    assert not _by_tiles(64, 4096, 65536, 4096, 4096, 1)
