"""A token of the vocabulary's size or more: log probability NaN, and the gradient of
the definition where no logit stands for the token, x_token - log sum e^x with a NaN
constant for x_token: -p times the cotangent.  A loss that leaves such positions out
or clips them gives a cotangent of 0 and with it a gradient of 0, not NaN."""
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [5, 4099])
def test_gradient_is_the_definitions(vocab):
    from pratchya_amd import functional as F
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn((4, vocab), generator=gen)
    tokens = torch.tensor([1, vocab, vocab + 7, 2 ** 40])
    g = torch.randn(4, generator=gen)
    u = x.double().requires_grad_(True)
    picked = u.gather(1, tokens.clamp(max=vocab - 1)[:, None])[:, 0]
    lp = torch.where(tokens < vocab, picked, math.nan) - torch.logsumexp(u, 1)
    want, = torch.autograd.grad(lp, u, g.double())
    xd = x.cuda().requires_grad_(True)
    got = F.token_logprobs(xd, tokens.cuda()).logprobs
    assert torch.isnan(got).tolist() == [False, True, True, True]
    dx, = torch.autograd.grad(got, xd, g.cuda())
    R.close(dx, want, torch.full_like(want, 256 * R.U * float(g.abs().max())), "dx")


@pytest.mark.parametrize("loss", [
    lambda lp: lp.nan_to_num(0.0).sum(), lambda lp: lp.nansum(), lambda lp: lp.clamp(min=-20).sum(),
    lambda lp: torch.where(torch.isnan(lp), 0.0, lp).sum(), lambda lp: lp[~torch.isnan(lp)].mean()])
def test_positions_left_out_have_no_gradient(loss):
    from pratchya_amd import functional as F
    x = torch.randn(6, 100, device="cuda", requires_grad=True)
    tokens = torch.tensor([3, 100, 5, 1000, -1, 7], device="cuda")
    dx, = torch.autograd.grad(loss(F.token_logprobs(x, tokens).logprobs), x)
    assert torch.equal(dx[[1, 3, 4]], torch.zeros_like(dx[[1, 3, 4]]))
    assert bool(torch.isfinite(dx).all()) and bool((dx[[0, 2, 5]].abs().sum(1) > 0).all())
