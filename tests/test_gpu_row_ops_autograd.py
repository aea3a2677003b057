"""What the row operators hold between the passes, and how their autograd nodes
behave: memory of 8-bit inputs, changed inputs, graphs used twice or freed, errors
of the library, other threads."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _F():
    from pratchya_amd import functional
    return functional


def _x(rows=64, width=1024, dtype=torch.bfloat16, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((rows, width), generator=gen).to(dtype).cuda()


def _held(call, rows=4096, width=4096):
    """Bytes an operator's output keeps alive beyond itself once its input is gone."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    leaf = torch.zeros((), device="cuda", requires_grad=True)
    x = _x(rows, width) + leaf.to(torch.bfloat16)
    y = call(x)
    size = x.numel() * 2
    del x
    held = torch.cuda.memory_allocated() - before - size
    y.float().sum().backward()
    assert leaf.grad is not None
    return held


@pytest.mark.parametrize("op", ["norm", "act"])
def test_eight_bits_are_held(op):
    F = _F()
    call = {"norm": lambda g: (lambda x: F.layer_norm(x, tgrid=g)),
            "act": lambda g: (lambda x: F.activation(x, "silu", tgrid=g))}[op]
    n = 4096 * 4096
    assert _held(call(None)) >= 2 * n
    # a byte an element, a byte a block, four bytes a group of eight blocks, a row's statistics
    assert _held(call((1, 128))) <= n + n // 128 + n // 256 + 8 * 4096 + (1 << 16)


def test_changed_input():
    """An input changed in place between the passes is refused where it is read again, and does not matter
    where its 8-bit form was kept."""
    F = _F()
    for call in (lambda x: F.layer_norm(x), lambda x: F.activation(x, "gelu"),
                 lambda x: F.token_logprobs(x, torch.zeros(64, dtype=torch.int64, device="cuda")).logprobs):
        x = _x().requires_grad_(True) * 1
        y = call(x)
        with torch.no_grad():
            x += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.float().sum().backward()
    leaf = _x().requires_grad_(True)
    want, = torch.autograd.grad(F.activation(leaf, "gelu", tgrid=(1, 32)).float().sum(), leaf)
    x = leaf * 1
    y = F.activation(x, "gelu", tgrid=(1, 32))
    with torch.no_grad():
        x += 1
    y.float().sum().backward()
    assert torch.equal(leaf.grad, want)


def test_graphs_used_twice_and_freed():
    F = _F()
    for tgrid in (None, (1, 128)):
        x = _x().requires_grad_(True)
        w = torch.ones(1024, device="cuda", requires_grad=True)
        y = F.layer_norm(x, w, tgrid=tgrid)
        g = _x(seed=2)
        first = torch.autograd.grad(y, (x, w), g, retain_graph=True)
        again = torch.autograd.grad(y, (x, w), g)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, (x, w), g)


def test_threads():
    """Passes of several threads at once, each with its own stream and data, give each its own bits."""
    F = _F()

    def work(seed):
        x = _x(300, 2048, seed=seed).requires_grad_(True)
        w = (1 + _x(1, 2048, torch.float32, seed + 50)[0] * 0.1).requires_grad_(True)
        y = F.activation(F.layer_norm(x, w, groups=16, tgrid=(1, 128)), "silu", tgrid=(1, 64))
        r = F.token_logprobs(y, torch.full((300,), seed, device="cuda"), entropy=True, top=9)
        return (r.logprobs, r.entropy, r.top_tokens) + torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), (x, w))
    want = [work(s) for s in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(s):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[s] = work(s)
            stream.synchronize()
        except BaseException as e:       # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_no_grad_and_leaves():
    F = _F()
    x = _x().requires_grad_(True)
    with torch.no_grad():
        assert F.layer_norm(x).grad_fn is None and F.activation(x).grad_fn is None
    assert F.layer_norm(x.detach()).grad_fn is None
    r = F.token_logprobs(x, torch.zeros(64, dtype=torch.int64, device="cuda"), entropy=True, top=3)
    assert r.logprobs.requires_grad and r.entropy.requires_grad and not r.top_logprobs.requires_grad
    r.entropy.sum().backward()               # one of two outputs
    assert x.grad is not None
    with torch.inference_mode():
        assert not F.layer_norm(_x()).requires_grad


def test_library_errors():
    """The library's refusals come as the framework's errors."""
    from pratchya_amd import _lib
    with pytest.raises(_lib.PratchyaUnsupported, match="2\\^20"):
        _F().layer_norm(torch.zeros((1, 1 << 21), device="cuda"), groups=1 << 21)


def test_stored_segments_of_eights():
    """A segment of an 8-bit input starts at a vector's boundary, so that no vector lies in two blocks or beyond
    the array: other segments are refused before any launch, by the binding and by the library."""
    from pratchya_amd import _kernels as K
    from pratchya_amd import _lib
    x = torch.zeros((4, 96), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="multiple of 8"):
        _F().layer_norm(x, groups=8, tgrid=(1, 32))
    stats = torch.zeros((32, 2), device="cuda")
    with pytest.raises(_lib.PratchyaUnsupported, match="not of eights"):
        K.layer_norm_bwd(K.quantize(x.detach(), (1, 32)), torch.zeros((4, 96), device="cuda"), None, stats, 8, (1, 32))
    y = _F().layer_norm(x, groups=4, tgrid=(1, 32))          # segments of 24
    y.sum().backward()
    assert x.grad is not None
