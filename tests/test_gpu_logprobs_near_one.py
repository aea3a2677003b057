"""token_logprobs where one token is nearly sure: no log probability is above 0 and no
entropy below 0, and a token that leaves the others less than 2^-26 has log
probability 0 to a rounding of 1, however the logits before it were ordered."""
import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
FORMS = [(300, 100), (40, 1000), (600, 4099), (20, 5003), (3, 70001)]


def _logits(rows, vocab, dt, lo, hi):
    """Normal logits with one standing out by lo to hi over the largest other, at any place of the row."""
    gen = torch.Generator().manual_seed(rows + vocab)
    x = torch.randn((rows, vocab), generator=gen)
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    x.scatter_(1, tokens[:, None], -100.0)
    best = x.amax(1) + torch.rand(rows, generator=gen) * (hi - lo) + lo
    return x.scatter_(1, tokens[:, None], best[:, None]).to(DT[dt]), tokens


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_sure_tokens(rows, vocab, dt, top):
    from pratchya_amd import functional as F
    for scale in (1.0, 3.0, 0.25):
        x, tokens = _logits(rows, vocab, dt, 32.0, 40.0)
        x = (x.float() * scale).to(DT[dt]) if scale > 1 else x
        x = x + 7 if scale < 1 else x
        r = F.token_logprobs(x.cuda(), tokens.cuda(), entropy=True, top=top)
        # the others hold at most vocab e^-32 < 2^-29: a sum of 1 and a logarithm of 0
        assert float(r.logprobs.max()) <= 0.0 and float(r.logprobs.min()) >= -R.U
        assert float(r.entropy.min()) >= 0.0 and float(r.entropy.max()) <= R.U + vocab * 2.0 ** -40
        if top:
            assert torch.equal(r.top_logprobs[:, 0], r.logprobs) and torch.equal(r.top_tokens[:, 0].cpu(), tokens)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_signs(rows, vocab, dt):
    """Any row: the token's own weight in the sum is 1 or less, the sum 1 or more."""
    from pratchya_amd import functional as F
    for lo, hi in ((0.0, 9.0), (6.0, 20.0)):
        x, tokens = _logits(rows, vocab, dt, lo, hi)
        r = F.token_logprobs(x.cuda(), tokens.cuda(), entropy=True, top=2)
        assert float(r.logprobs.max()) <= 0.0 and float(r.entropy.min()) >= 0.0
        assert float(r.top_logprobs.max()) <= 0.0
        n = F.token_logprobs(x.cuda(), tokens.cuda(), entropy=True)
        assert float(n.logprobs.max()) <= 0.0 and float(n.entropy.min()) >= 0.0


@pytest.mark.parametrize("vocab", [100, 1000, 20000])
def test_as_exact_as_the_plain_form(vocab):
    """Log probabilities near 0 against 64 bits: on average no more than twice as far off as log_softmax in 32
    bits, whose largest term is 1 exactly."""
    from pratchya_amd import functional as F
    x, tokens = _logits(2000, vocab, "f32", 5.0, 12.0)
    want = torch.log_softmax(x.double(), 1).gather(1, tokens[:, None])[:, 0]
    d = x - x.amax(1, keepdim=True)
    plain = (d - torch.log(torch.exp(d).sum(1, keepdim=True))).gather(1, tokens[:, None])[:, 0]
    got = F.token_logprobs(x.cuda(), tokens.cuda()).logprobs.cpu()
    off = (got.double() - want).abs().mean()
    assert float(off) <= 2 * float((plain.double() - want).abs().mean()) + 0.5 * R.U


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [200, 520])
@pytest.mark.parametrize("vocab", [2000, 20000])
def test_a_larger_logit_later(rows, vocab, dt, top):
    """The token's logit comes after one or more that are a few units smaller, at places that one thread reads one
    after the other; all others are far below.  Bounds: the sum, below 4, is rounded with each of them (U times 2
    at most, over a sum of 1 or more), their powers carry a few U of themselves, the logarithm of itself."""
    from pratchya_amd import functional as F
    n = 8 if dt == "bf16" else 4
    gen = torch.Generator().manual_seed(rows + vocab)
    x = torch.full((rows, vocab), -60.0)
    steps = [64 * n] if vocab < 1025 * n else [64 * n, 256 * n, 1024 * n]
    tokens = torch.randint(steps[-1], vocab, (rows,), generator=gen)
    # eighths, exact in both types: the gaps are what they are said to be
    last = torch.randint(-40, 40, (rows,), generator=gen) / 8
    gap = torch.randint(4, 64, (rows,), generator=gen) / 8
    x.scatter_(1, tokens[:, None], last[:, None])
    for s in steps:
        x.scatter_(1, (tokens - s)[:, None], (last - gap)[:, None])
    q = len(steps) * torch.exp(-gap.double())
    r = F.token_logprobs(x.to(DT[dt]).cuda(), tokens.cuda(), entropy=True, top=top)
    want = -torch.log1p(q)
    bound = (2 * len(steps) + q * (8 + 2 * gap) + 2 * want.abs()) * R.U
    R.close(r.logprobs, want, bound, "logprobs")
    p = torch.exp(want)
    H = -want + q * p * gap
    R.close(r.entropy, H, 2 * bound + q * p * gap * (16 + 2 * gap) * R.U, "entropy")
