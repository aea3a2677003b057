"""Backward passes of several threads through one graph of embedding, linear attention and the
head's cross entropy: with the graph retained all get the same bits; without, each gets them or
torch's error that the graph is gone.  Also two graphs of the same leaves captured one after
the other and replayed in turn, whose workspaces are their own."""
import pytest
import torch

from tests.test_gpu_row_ops_shared_graph import _together

pytestmark = pytest.mark.gpu


def _leaves(seed):
    gen = torch.Generator().manual_seed(seed)
    table = torch.randn((1000, 512), generator=gen).to(torch.bfloat16).cuda().requires_grad_(True)
    slow = (-torch.rand(8, generator=gen)).cuda().requires_grad_(True)
    tokens = torch.randint(-1, 1000, (2, 400), generator=gen).cuda()
    return table, slow, tokens


def _loss(table, slow, tokens):
    from pratchya_amd import functional as F
    x = F.embedding(table, tokens, scale=0.2)
    q = x.unflatten(-1, (8, 64))
    r = F.linear_attention(q, q, q, slow.expand(*tokens.shape, 8), scale=0.125)
    return F.linear_cross_entropy(r.out.flatten(2), table.t(), tokens).sum() + 0.01 * r.state.sum()


@pytest.mark.parametrize("retain", [True, False])
def test_shared(retain):
    table, slow, tokens = _leaves(1)
    want = torch.autograd.grad(_loss(table, slow, tokens), (table, slow))
    for _ in range(10):
        loss = _loss(table, slow, tokens)
        got = _together(4, lambda: torch.autograd.grad(loss, (table, slow), retain_graph=retain))
        whole = [g for g in got if isinstance(g, tuple)]
        assert len(whole) == 4 if retain else whole
        for g in got:
            if isinstance(g, tuple):
                assert all(torch.equal(a, b) for a, b in zip(g, want))
            else:
                assert "second time" in str(g)


def test_two_graphs():
    table, slow, tokens = _leaves(2)
    other = tokens.flip(1).contiguous()
    for t in (tokens, other):
        torch.autograd.grad(_loss(table, slow, t), (table, slow))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in (tokens, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(torch.autograd.grad(_loss(table, slow, t), (table, slow)))
        graphs.append(graph)
    for rep in range(3):
        with torch.no_grad():
            table.add_(0.01 * torch.randn_like(table))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        want = [torch.autograd.grad(_loss(table, slow, t), (table, slow)) for t in (tokens, other)]
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w)), rep
