"""What stands around and between the quantized Linears of a model: embedding, layer
norm, activations, linear attention, the log probabilities of tokens over the head's
logits, and the head's cross entropy without logits, each with its gradients, on the
gfx950 kernels.

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

A language model with tied weights and linear attention begins, mixes and ends with

    x = functional.embedding(table, tokens, scale=C ** 0.5)
    r = functional.linear_attention(q, k, v, log_decay, lengths=lengths, scale=D ** -0.5)
    loss = functional.linear_cross_entropy(x, table.t(), targets)

and generates with ``linear_attention_step`` from ``r.state`` on.

Arrays are bf16 or f32 on the GPU; rows may be a stride apart (slices of a wider
array).  Arithmetic is f32, with one rounding to a result's type; where values between
have fewer bits, the operator says so.  Gradients are reverse-mode and of first order: inputs with a forward-mode tangent are refused, and
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


def embedding(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[tokens]`` for a table [V, C] and tokens [...] (int64 or int32),
    [..., C] in the table's dtype, differentiable in the table: its gradient is dense,
    f32 sums over a token's occurrences in their order, rounded once.

    A negative token stands for none: its row is 0 and it has no gradient.  A token of V
    or more gives NaN, as no row stands for it, and has no gradient."""
    return _ops.embedding(table, tokens, scale)


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


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         label_smoothing: float = 0.0) -> torch.Tensor:
    """Softmax cross entropy of the output head ``z = x @ weight``, for x [..., C],
    weight [C, V] of x's dtype and targets [...] (int64 or int32): f32 [...],
    ``(1 - a) (lse - z_t) + a (lse - mean z)`` with a the label smoothing,
    differentiable in x and weight.  The logits are not kept: both passes compute them,
    in f32, by tiles or a piece of the vocabulary at a time; their gradient, likewise, is
    rounded to x's dtype before the products that give the gradients of x and weight.  In
    bf16 the gradients' error is then that of their own rounding (0.0017 of the norm) with
    thousands of rows, and up to 1.4 times that with few rows and a small vocabulary.  An
    embedding table [V, C] serves as weight through its transposed view ``table.t()``,
    which is read as it lies.

    A negative target stands for none: its loss is 0 and has no gradient.  A target of V
    or more gives NaN, as no logit stands for it; its gradient is that of the other
    terms.  A row of x that holds a NaN or an infinity has a loss and a gradient that are
    not finite, and so is the weight's gradient unless the row has no target; the other
    rows' are not touched."""
    return _ops.linear_cross_entropy(x, weight, targets, label_smoothing)


class LinearAttention(NamedTuple):
    """Results of ``linear_attention``."""
    out: torch.Tensor                           # [B, T, H, E], of q's dtype
    state: torch.Tensor                         # f32 [B, H, D, E]


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                     scale: float = 1.0) -> LinearAttention:
    """Linear attention with a decay for each head and token: with a state S [D, E] per
    sequence and head,

        S_t = exp(log_decay_t) S_(t-1) + k_t^T v_t,      out_t = scale * q_t S_t

    for q, k [B, T, H, D] and v [B, T, H, E] (bf16 or f32, heads of up to 128, rows at
    any strides) and log_decay [B, T, H] (bf16 or f32; decays that are the same for all
    tokens are an expanded array; -inf forgets all).  ``state`` is S before the first
    token, f32 [B, H, D, E], or None for 0; the result holds S behind the last one.
    Differentiable in all of them, states included.

    ``lengths`` [B] (int64 or int32): tokens from a sequence's length on are padding.
    They are not read, their outputs and gradients are 0, and the state is that behind
    the last token before them.  A NaN or an infinity reaches the results that the
    recurrence takes it to, there as one or the other; in gradients of log_decay, sums
    over later tokens, it reaches earlier tokens too.  States are f32; where results in bf16 read them, and for
    the scores of tokens with each other, 16 bits of their values count.  Long sequences are cut into
    segments, into more of them where no gradient is recorded: the results then differ in
    roundings."""
    return LinearAttention(*_ops.linear_attention(q, k, v, log_decay, state, lengths, scale))


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """One token of ``linear_attention`` for each sequence: q, k [B, H, D], v [B, H, E],
    log_decay [B, H]; ``state`` (f32 [B, H, D, E], contiguous) is updated in place, and
    the result is [B, H, E].  For generation: it has no gradient."""
    return _ops.linear_attention_step(q, k, v, log_decay, state, scale)
