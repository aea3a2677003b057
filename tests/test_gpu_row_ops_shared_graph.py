"""Backward passes of several threads through one graph of the row operators: with the
graph retained all get the same bits; without, each gets them or torch's error that
the graph is gone.  Also from hooks, where a thread of torch's own runs the pass."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _graph(seed):
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((64, 1024), generator=gen).to(torch.bfloat16).cuda().requires_grad_(True)
    w = (1 + 0.1 * torch.randn(1024, generator=gen)).cuda().requires_grad_(True)
    y = F.activation(F.layer_norm(x, w, groups=8, tgrid=(1, 64)), "silu", tgrid=(1, 128))
    r = F.token_logprobs(F.layer_norm(y, w), torch.arange(64, device="cuda"), entropy=True)
    return r.logprobs.sum() + r.entropy.sum(), (x, w)


def _together(n, body):
    """body() in n threads that start together: their results, or the errors they raised."""
    out, gate = [None] * n, threading.Barrier(n)

    def run(i):
        gate.wait()
        try:
            out[i] = body()
        except RuntimeError as e:
            out[i] = e
    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("retain", [True, False])
def test_shared(retain):
    loss, leaves = _graph(1)
    want = torch.autograd.grad(loss, leaves)
    for _ in range(20):
        loss, leaves = _graph(1)
        got = _together(4, lambda: torch.autograd.grad(loss, leaves, retain_graph=retain))
        whole = [g for g in got if isinstance(g, tuple)]
        assert len(whole) == 4 if retain else whole
        for g in got:
            if isinstance(g, tuple):
                assert all(torch.equal(a, b) for a, b in zip(g, want))
            else:
                assert "second time" in str(g)


def test_from_a_hook():
    """A backward pass inside another one's hook, of the same graph."""
    loss, leaves = _graph(2)
    want = torch.autograd.grad(loss, leaves, retain_graph=True)
    inner = []
    leaves[0].register_hook(lambda g: inner.append(torch.autograd.grad(loss, leaves[1], retain_graph=True)) or None)
    got = torch.autograd.grad(loss, leaves, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert len(inner) == 1 and torch.equal(inner[0][0], want[1])
