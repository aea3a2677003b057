"""The operators together, as examples/train_and_score.py runs them: the loss falls,
the scores agree with plain torch on the same logits, and a step's gradients with
those of the same model whose norms, activation and loss are plain torch."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "train_and_score.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_and_score", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_runs(example):
    p, losses, scores = example.main(steps=25)
    assert bool(torch.isfinite(losses).all())
    assert float(losses[-5:].mean()) < 0.8 * float(losses[:5].mean())
    tokens, targets = example.batch(512, 8, -1)
    with torch.no_grad():
        lp = torch.log_softmax(example.logits(p, tokens).double(), dim=1)
    want = torch.where(targets < 0, 0.0, lp.gather(1, targets.clamp(min=0)[:, None])[:, 0])
    assert float((scores.logprobs.double() - want).abs().max()) < 1e-4
    assert float((scores.entropy.double() + (lp.exp() * lp).sum(1)).abs().max()) < 1e-4
    assert float((scores.top_logprobs[:, 0].double() - lp.max(dim=1).values).abs().max()) < 1e-4


def test_gradients_of_a_step(example, monkeypatch):
    """8-bit inputs change a norm's or activation's gradient by e4m3's step, 2^-4 of a value at most; through the
    whole model the gradients stay within a tenth of those of plain torch around the same quantized Linears."""
    p = example.init(512, 1024, 2048, seed=3)
    tokens, targets = example.batch(512, 512, 1)
    leaves = [t for v in p.values() for t in (v if isinstance(v, list) else [v])]

    def grads():
        out = example.F.token_logprobs(example.logits(p, tokens), targets, entropy=True)
        return torch.autograd.grad(-out.logprobs.sum() / 480 - 0.001 * out.entropy.mean(), leaves)
    got = grads()

    class Plain:
        TokenLogprobs = example.F.TokenLogprobs

        @staticmethod
        def layer_norm(x, w, b, eps=1e-5, groups=1, tgrid=None):
            seg = x.float().reshape(x.shape[0], groups, -1)
            h = (seg - seg.mean(2, keepdim=True)) / (seg.var(2, correction=0, keepdim=True) + eps).sqrt()
            return (h.reshape(x.shape) * w + b).to(x.dtype)

        @staticmethod
        def activation(x, kind, tgrid=None):
            return (x.float().clamp(min=0) ** 2).to(x.dtype)

        @staticmethod
        def token_logprobs(x, t, entropy, top=0):
            lp = torch.log_softmax(x.float(), dim=1)
            tok = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
            return example.F.TokenLogprobs(tok, -(lp.exp() * lp).sum(1), None, None)
    monkeypatch.setattr(example, "F", Plain)
    want = grads()
    for g, w in zip(got, want):
        assert float((g.float() - w.float()).norm() / w.float().norm()) < 0.1
