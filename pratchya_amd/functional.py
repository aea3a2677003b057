"""What stands between the quantized Linears of a model: layer norm,
activations, and the log probabilities of tokens over the head's logits, each
with its gradients, on the gfx950 kernels.

``layer_norm`` and ``activation`` can keep their input for the backward pass in
8 bits (``tgrid=(1, b)``): the forward pass quantizes it as
``qarr.quantize_impl(x.reshape(-1, C), tgrid)`` does and computes its result
from x itself; the backward pass reads the quantized form.  That is one byte an
element (and the blocks' scales) instead of two or four held from the forward
to the backward pass, as the quantized Linear holds its own input.

    h = functional.layer_norm(x, w, b, tgrid=(1, 128))
    u = (QArrayImpl(h, (1, 128)) @ up).astype(h.dtype)
    x = x + (QArrayImpl(functional.activation(u, "relu2", tgrid=(1, 128)), (1, 128)) @ down).astype(x.dtype)
    loss = -functional.token_logprobs(logits, tokens).logprobs.mean()

Arrays are bf16 or f32 on the GPU; rows may be a stride apart (slices of a wider
array).  Arithmetic is f32, with one rounding to a result's type.  Gradients are
reverse-mode and of first order: inputs with a forward-mode tangent are refused, and
so is the gradient of a gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _kernels as K
from . import _lib

_ops = _lib.row_ops()


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, groups: int = 1, tgrid: Optional[Tuple[int, int]] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of x
    [..., C], or over each of ``groups`` equal segments of it (the heads of a norm
    over heads); weight and bias [C] or None.  With ``tgrid=(1, b)``, b 16, 32, 64 or
    128 dividing C, and segments of a multiple of 8 elements, x is kept for the
    backward pass in 8 bits with that block grid (its mean and deviation in f32, of
    x itself).  Without a gradient to
    compute nothing is kept, and ``tgrid`` has no effect."""
    return _ops.layer_norm(x, weight, bias, eps, groups, tgrid)


def activation(x: torch.Tensor, kind: str = "relu2", tgrid: Optional[Tuple[int, int]] = None) -> torch.Tensor:
    """``max(x, 0)^2`` ("relu2"), ``x / (1 + exp(-x))`` ("silu") or x times the
    normal distribution function of x ("gelu"), for x [..., C].  With
    ``tgrid=(1, b)``, b 16, 32, 64 or 128 dividing C, x is kept for the backward
    pass in 8 bits with that block grid; without a gradient to compute it has no
    effect."""
    return _ops.activation(x, K._activation_code(kind), tgrid)


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``; what was not asked for is None."""
    logprobs: torch.Tensor                      # f32 [...]
    entropy: Optional[torch.Tensor]             # f32 [...]
    top_logprobs: Optional[torch.Tensor]        # f32 [..., top]
    top_tokens: Optional[torch.Tensor]          # int64 [..., top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, entropy: bool = False, top: int = 0) -> TokenLogprobs:
    """Log probability of ``tokens`` [...] (int64 or int32) under softmax of
    ``logits`` [..., V], with ``entropy`` the distributions' entropy, and with
    ``top`` (up to 64) the most probable tokens and their log probabilities, in
    falling order, equal logits by index.  Log probabilities and entropy are
    differentiable in the logits, the alternatives are not.

    A negative token stands for none: its log probability is 0 and has no
    gradient.  A token of V or more gives NaN, as no logit stands for it; its gradient
    is that of the sum alone, -p times the cotangent, so a position that the loss leaves
    out (``nansum``, ``where``, ``clamp``) has none.  Logits of -inf are masked; a row of
    nothing else has log probabilities of -inf and entropy 0, and in its gradient,
    as for any masked logit, the probability 0."""
    return TokenLogprobs(*_ops.token_logprobs(logits, tokens, entropy, top))
