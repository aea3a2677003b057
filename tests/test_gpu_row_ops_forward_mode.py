"""Forward-mode derivatives of the row operators are refused, not dropped: an output
without a tangent would stand for a derivative of 0."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def _calls():
    from pratchya_amd import functional as F
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    w = torch.ones(64, device="cuda")
    return {"layer_norm": lambda t: F.layer_norm(t), "groups": lambda t: F.layer_norm(t, w, w, groups=4),
            "activation": lambda t: F.activation(t, "silu"), "stored": lambda t: F.activation(t, "relu2", tgrid=(1, 32)),
            "token_logprobs": lambda t: F.token_logprobs(t, tok, entropy=True, top=2)}


@pytest.mark.parametrize("name", ["layer_norm", "groups", "activation", "stored", "token_logprobs"])
@pytest.mark.parametrize("grad", [False, True])
def test_refused(name, grad):
    call = _calls()[name]
    x = torch.randn(4, 64, device="cuda").requires_grad_(grad)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwd.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwd.make_dual(x.detach(), torch.ones_like(x)))
        call(x)                       # without a tangent: as ever
    call(x)


def test_parameters():
    from pratchya_amd import functional as F
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with fwd.dual_level():
        d = fwd.make_dual(w, w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            F.layer_norm(x, d)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            F.layer_norm(x, None, d)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: F.activation(t, "gelu"), (x,), (x,))
