"""A gradient of the row operators cannot be differentiated again: with create_graph it
leads into an error, also in a sum with parts that can, where it would count as a
constant otherwise."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    from pratchya_amd import functional as F
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    return {"layer_norm": lambda t: F.layer_norm(t), "activation": lambda t: F.activation(t, "silu"),
            "stored": lambda t: F.activation(t, "gelu", tgrid=(1, 32)),
            "token_logprobs": lambda t: F.token_logprobs(t, tok).logprobs, "embedding": lambda t: F.embedding(t, tok)}


@pytest.mark.parametrize("name", ["layer_norm", "activation", "stored", "token_logprobs", "embedding"])
def test_twice(name):
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    call = _calls()[name]
    once, = torch.autograd.grad(call(x).sum(), x)
    g, = torch.autograd.grad(call(x).sum(), x, create_graph=True)
    assert torch.equal(g, once)
    with pytest.raises(RuntimeError, match="again"):
        (g.sum() + (x * x).sum()).backward()
