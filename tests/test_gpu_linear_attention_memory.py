"""What linear_attention holds between its passes: the states before the segments, not those of
their parts; and the C entry that takes both in one array gives the same bits."""
import pytest
import torch

from tests.test_gpu_linear_attention import _F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_held_for_the_backward_pass(dtype):
    from pratchya_amd import _lib
    B, T, H, D = 1, 8192, 8, 64
    q, k, v = (torch.randn((B, T, H, D), device="cuda", dtype=dtype).requires_grad_(True) for _ in range(3))
    g = torch.full((B, T, H), -0.05, device="cuda")
    _F().linear_attention(q, k, v, g)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    r = _F().linear_attention(q, k, v, g)
    held = torch.cuda.memory_allocated() - before
    args = (B, T, H, D, D, int(dtype == torch.bfloat16), 1)
    kept = _lib.load().pratchya_linear_attention_states_floats(*args)
    assert 0 < kept < _lib.load().pratchya_linear_attention_starts_floats(*args)
    results = r.out.numel() * r.out.element_size() + r.state.numel() * 4
    assert held <= results + 4 * kept + 3 * 2 ** 20      # the allocator's granules
    assert 4 * kept + 3 * 2 ** 20 < 4 * _lib.load().pratchya_linear_attention_starts_floats(*args)


def test_both_entries():
    import ctypes
    from pratchya_amd import _lib
    lib = _lib.load()
    B, T, H, D = 1, 2000, 4, 32
    q, k, v = (torch.randn((B, T, H, D), device="cuda") for _ in range(3))
    g = -torch.rand((B, T, H), device="cuda")
    strides = (ctypes.c_int64 * 12)(*[s for t in (q, k, v, g) for s in t.stride()[:3]])
    floats = lib.pratchya_linear_attention_starts_floats(B, T, H, D, D, 0, 1)
    kept = lib.pratchya_linear_attention_states_floats(B, T, H, D, D, 0, 1)
    assert 0 < kept < floats

    def call(entry, *space):
        out, state = torch.empty_like(v), torch.empty((B, H, D, D), device="cuda")
        assert entry(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, g.data_ptr(), 0, strides, None, None, B, T, H, D, D, 0.5, 1,
                     out.data_ptr(), state.data_ptr(), *[s.data_ptr() for s in space],
                     torch.cuda.current_stream().cuda_stream) == _lib.OK
        torch.cuda.synchronize()
        return out, state
    whole, starts, parts = (torch.empty(n, device="cuda") for n in (floats, kept, floats - kept))
    a, b = call(lib.pratchya_linear_attention, whole), call(lib.pratchya_linear_attention_parts, starts, parts)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(whole[:kept], starts)
