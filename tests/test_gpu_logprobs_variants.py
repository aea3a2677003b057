"""token_logprobs on both sides of every size at which another kernel variant runs:
512 rows, 2048 logits, the arrays that are read or written past the caches (forward
above 256 MB, backward above 32 MB), remainders of vectors and pieces, 32 and 33
alternatives; entropies, both cotangents, masks and missing tokens in each."""
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(rows, vocab, dt, entropy=True, every=1):
    """Through autograd on the GPU; rows 0, every, 2 every ... and the last against the 64-bit form."""
    from pratchya_amd import functional as F
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = torch.randn((rows, vocab), generator=gen, device="cuda", dtype=DT[dt]).mul_(2.5)
    x[:, vocab - vocab // 50:] = -math.inf
    x[1::7, : vocab // 2] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    tokens[::5] = -1
    tokens[rows - 1] = vocab - vocab // 2 - 1
    x[rows // 2] = -math.inf                                     # nothing left
    g, gh = (torch.randn(rows, generator=gen, device="cuda") for _ in range(2))
    x.requires_grad_(True)
    r = F.token_logprobs(x, tokens, entropy=entropy)
    ends, cots = ((r.logprobs, r.entropy), (g, gh)) if entropy else ((r.logprobs,), (g,))
    dx, = torch.autograd.grad(ends, x, cots)
    at = sorted(set(range(0, rows, every)) | {1, rows // 2, rows - 1})
    pick = torch.tensor(at, device="cuda")
    want, bound = R.token_logprobs(x.detach()[pick].cpu(), tokens[pick].cpu(), g[pick].cpu(),
                                   gh[pick].cpu() if entropy else None)
    R.close(r.logprobs[pick], want[0], bound[0], "logprobs")
    if entropy:
        R.close(r.entropy[pick], want[1], bound[1], "entropy")
    R.close(dx[pick], want[2], bound[2], "dx")
    # every row, whether compared above or not
    assert bool(torch.isfinite(dx).all())
    plain = F.token_logprobs(x.detach(), tokens, entropy=entropy)
    assert torch.equal(plain.logprobs, r.logprobs) and (not entropy or torch.equal(plain.entropy, r.entropy))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("entropy", [True, False])
@pytest.mark.parametrize("rows", [511, 512, 600])
@pytest.mark.parametrize("vocab", [2047, 2048, 2049, 4099, 5003])
def test_rows_and_vocabularies(rows, vocab, entropy, dt):
    _case(rows, vocab, dt, entropy, 7)


@pytest.mark.parametrize("rows,vocab,dt", [(1310, 13001, "bf16"), (610, 14003, "f32"), (2050, 16384, "bf16"),
                                           (700, 50021, "f32"), (1290, 13001, "bf16"), (590, 14003, "f32")])
def test_gradients_past_the_caches(rows, vocab, dt):
    """Around 32 MB of logits, with whole and partial pieces."""
    _case(rows, vocab, dt, True, 131)


@pytest.mark.parametrize("rows,vocab,dt,entropy", [(2700, 50021, "bf16", True), (1400, 50021, "f32", True),
                                                   (2700, 50021, "bf16", False), (1400, 50021, "f32", False),
                                                   (2100, 65536, "bf16", True)])
def test_logits_past_the_caches(rows, vocab, dt, entropy):
    """More than 256 MB of logits."""
    _case(rows, vocab, dt, entropy, 499)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(5, 33), (6, 64), (4, 4096), (3, 4097), (5, 20001), (600, 2100)])
@pytest.mark.parametrize("top", [31, 32, 33, 34])
def test_alternatives_around_32(rows, vocab, top, dt):
    from pratchya_amd import functional as F
    top = min(top, vocab)
    gen = torch.Generator().manual_seed(rows + vocab + top)
    x = torch.randn((rows, vocab), generator=gen).to(DT[dt])
    x[rows // 2] = (x[rows // 2] * 2).round()                    # many equal values
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    r = F.token_logprobs(x.cuda(), tokens.cuda(), top=top)
    best = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_tokens.cpu(), best)
    for k in (0, top // 2, top - 1):
        want, bound = R.token_logprobs(x, best[:, k])
        R.close(r.top_logprobs[:, k], want[0], bound[0], f"alternative {k}")
