"""The operators together, as examples/linear_attention_lm.py runs them: a step's gradients
agree with those of the same model in plain torch around the same quantized Linears, tokens
one by one with the whole sequence, and a captured step with the eager one."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "linear_attention_lm.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("linear_attention_lm", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_runs(example):
    p, losses, tokens = example.main(steps=3)
    assert losses.shape == (3,) and bool(torch.isfinite(losses).all())
    assert tokens.shape == (4, 6) and bool(((tokens >= 0) & (tokens < 512)).all())
    assert all(bool(torch.isfinite(t).all()) for t in example.leaves(p))


class Plain:
    """The operators in elementary torch operations, results rounded to the inputs' type."""

    @staticmethod
    def embedding(table, tokens, scale=1.0):
        return (table[tokens].float() * scale).to(table.dtype)

    @staticmethod
    def layer_norm(x, w, b, eps=1e-5, groups=1, tgrid=None):
        seg = x.float().reshape(x.shape[0], groups, -1)
        h = (seg - seg.mean(2, keepdim=True)) / (seg.var(2, correction=0, keepdim=True) + eps).sqrt()
        return (h.reshape(x.shape) * w + b).to(x.dtype)

    @staticmethod
    def linear_attention(q, k, v, log_decay, state=None, lengths=None, scale=1.0):
        B, T, H, D = q.shape
        S, out = torch.zeros((B, H, D, v.shape[-1]), device=q.device), []
        for t in range(T):
            live = (t < lengths).float()[:, None, None, None]
            new = torch.exp(log_decay[:, t])[..., None, None] * S + k[:, t].float()[..., :, None] * v[:, t].float()[..., None, :]
            S = live * new + (1 - live) * S
            out.append(live[..., 0] * scale * (q[:, t].float()[..., :, None] * S).sum(-2))

        class R:
            pass
        R.out, R.state = torch.stack(out, 1).to(q.dtype), S
        return R

    @staticmethod
    def linear_cross_entropy(x, w, targets, label_smoothing=0.0):
        lp = torch.log_softmax(x.float() @ w.float(), -1)
        loss = -(1 - label_smoothing) * lp.gather(-1, targets.clamp(min=0)[..., None])[..., 0] - label_smoothing * lp.mean(-1)
        return torch.where(targets < 0, 0.0, loss)


def test_gradients_of_a_step(example, monkeypatch):
    """Through the quantized Linears, whose 8 bits (steps of 2^-4) turn on differences of a rounding of
    bf16, the gradients stay within a tenth of each other."""
    p = example.init(512, 512, seed=3)
    tokens, targets, lengths = example.batch(512, 6, 70, 1)

    def grads():
        loss = example.losses(p, tokens, targets, lengths)
        return [loss] + list(torch.autograd.grad(loss.sum() / 100, example.leaves(p)))
    got = [t.detach() for t in grads()]
    monkeypatch.setattr(example, "F", Plain)
    want = [t.detach() for t in grads()]
    assert not bool(got[0][targets < 0].any())
    for g, w in zip(got, want):
        assert float((g.float() - w.float()).norm() / w.float().norm()) < 0.1


def test_tokens_one_by_one(example, monkeypatch):
    """Rows of the head from steps in place, from pieces, and from the whole sequences.  The quantized
    Linears' groups of 1024 values reach over rows of 512, so their 8 bits depend on a row's neighbours
    (4.9% of a row's norm between the same rows alone and among others); here they are plain products.
    What is left are roundings to bf16: of scores, states and outputs of the attention, three times
    2^-8 of sums of magnitudes that are a few times a row's, behind them two norms and the projection."""
    monkeypatch.setattr(example, "linear", lambda x, w: (x.float() @ w.float()).to(x.dtype))
    p = example.init(512, 512, seed=4)
    tokens, _, _ = example.batch(512, 3, 90, 2, back=5)
    with torch.no_grad():
        whole, last = example.hidden_rows(p, tokens)
        head, state = example.hidden_rows(p, tokens[:, :31])
        rows = [head]
        for t in range(31, 90):
            rows.append(example.step_rows(p, tokens[:, t], state)[:, None])
    both = torch.cat(rows, 1).float() - whole.float()
    assert float((both.norm(dim=-1) / whole.float().norm(dim=-1)).max()) < 12 * 2.0 ** -8
    assert float((state - last).norm() / last.norm()) < 500 * 2.0 ** -24


def test_captured_step(example):
    """Forward and backward passes of the whole model in one graph, replayed on new tokens between eager steps."""
    p = example.init(512, 512, seed=5)
    tokens, targets, lengths = example.batch(512, 4, 130, 0)

    def work():
        loss = example.losses(p, tokens, targets, lengths)
        return [loss] + list(torch.autograd.grad(loss, example.leaves(p), torch.full_like(loss, 1 / 400)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for step in range(1, 4):
        for old, new in zip((tokens, targets, lengths), example.batch(512, 4, 130, step)):
            old.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert math.isfinite(float(out[0].sum()))
        assert all(torch.equal(a, b) for a, b in zip(out, work())), step


def test_generation_in_a_graph(example):
    """One step of generation captured once: the state is carried by the buffer that it updates."""
    p = example.init(512, 512, seed=6)
    tokens, _, lengths = example.batch(512, 5, 40, 0)
    with torch.no_grad():
        _, state = example.hidden_rows(p, tokens, lengths)
        eager, token = state.clone(), tokens[:, 0].clone()
        example.step_rows(p, token, state.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        start = state.clone()
        with torch.cuda.graph(graph):
            row = example.step_rows(p, token, state)
        state.copy_(start)
        for t in range(4):
            token.copy_(tokens[:, t])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = example.step_rows(p, token, eager)
            assert torch.equal(row, want) and torch.equal(state, eager), t
