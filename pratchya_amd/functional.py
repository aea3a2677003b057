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
array).  Arithmetic is f32, with one rounding to a result's type.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _kernels as K


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, groups, tgrid):
        need = ctx.needs_input_grad
        y, stats, stored = K.layer_norm(x, weight, bias, eps, groups, True, tgrid if need[0] or need[1] else None)
        ctx.groups, ctx.tgrid = groups, None if stored is None else tgrid
        ctx.bias_dtype = torch.float32 if bias is None else bias.dtype
        ctx.save_for_backward(weight, stats, *((x,) if stored is None else stored))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, stats, *x = ctx.saved_tensors
        grads = K.layer_norm_bwd(x[0] if ctx.tgrid is None else x, dy, weight, stats, ctx.groups, ctx.tgrid,
                                 ctx.needs_input_grad[:3], ctx.bias_dtype)
        return grads + (None, None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, groups: int = 1, tgrid: Optional[Tuple[int, int]] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of x
    [..., C], or over each of ``groups`` equal segments of it (the heads of a norm
    over heads); weight and bias [C] or None.  With ``tgrid=(1, b)``, b 16, 32, 64 or
    128 dividing C, x is kept for the backward pass in 8 bits with that block
    grid (its mean and deviation in f32, of x itself)."""
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, groups, tgrid)
    return K.layer_norm(x, weight, bias, eps, groups)[0]


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, tgrid):
        y, stored = K.activation(x, kind, tgrid)
        ctx.kind, ctx.tgrid = kind, tgrid
        ctx.save_for_backward(*((x,) if stored is None else stored))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x = ctx.saved_tensors
        return K.activation_bwd(x[0] if ctx.tgrid is None else x, dy, ctx.kind, ctx.tgrid), None, None


def activation(x: torch.Tensor, kind: str = "relu2", tgrid: Optional[Tuple[int, int]] = None) -> torch.Tensor:
    """``max(x, 0)^2`` ("relu2"), ``x / (1 + exp(-x))`` ("silu") or x times the
    normal distribution function of x ("gelu"), for x [..., C].  With
    ``tgrid=(1, b)``, b 16, 32, 64 or 128 dividing C, x is kept for the backward
    pass in 8 bits with that block grid."""
    if torch.is_grad_enabled() and x.requires_grad:
        return _Activation.apply(x, kind, tgrid)
    return K.activation(x, kind)[0]


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``; what was not asked for is None."""
    logprobs: torch.Tensor                      # f32 [...]
    entropy: Optional[torch.Tensor]             # f32 [...]
    top_logprobs: Optional[torch.Tensor]        # f32 [..., top]
    top_tokens: Optional[torch.Tensor]          # int64 [..., top]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, entropy, top):
        logprobs, ent, top_lp, top_tok, stats = K.token_logprobs(logits, tokens, entropy, top, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (top_lp, top_tok) if t is not None))
        return logprobs, ent, top_lp, top_tok

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_entropy, *_):
        if g is None and g_entropy is None:
            return None, None, None, None
        return K.token_logprobs_bwd(*ctx.saved_tensors, g, g_entropy), None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, entropy: bool = False, top: int = 0) -> TokenLogprobs:
    """Log probability of ``tokens`` [...] (int64 or int32) under softmax of
    ``logits`` [..., V], with ``entropy`` the distributions' entropy, and with
    ``top`` (up to 64) the most probable tokens and their log probabilities, in
    falling order, equal logits by index.  Log probabilities and entropy are
    differentiable in the logits, the alternatives are not.

    A negative token stands for none: its log probability is 0 and has no
    gradient.  A token of V or more gives NaN.  Logits of -inf are masked; a row of nothing
    else has log probabilities of -inf, entropy 0 and no gradient."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, entropy, top))
    return TokenLogprobs(*K.token_logprobs(logits, tokens, entropy, top)[:4])
