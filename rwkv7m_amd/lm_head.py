"""Operators around a language model's head.

The end of the model and what is made of its logits:

* ``layer_norm``: the norm before the head, as before each block's mixes;
* ``token_logprobs``: log probabilities of given tokens, entropy and the top
  alternatives, for scoring, for a decode step's report and, being
  differentiable, for training on them;
* ``distill_loss``: the distillation loss from a teacher's top logits, whose
  gradient is formed in the same pass over the logits.

The head's product between the first and the other two is a plain GEMM and
stays the caller's (``x @ head.T``).  Each is one or two HIP kernels
(``kernels/lm_head_hip.py``); tensors are on the GPU, activations and logits
bf16 or fp32, and every sum is held in fp32 or more.  Gradients are first
order: a second derivative raises.  ``examples/distill_and_score.py`` runs
the three together.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .kernels import lm_head_hip


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in tensors)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = lm_head_hip.layer_norm_forward(x, weight, bias, eps,
                                                       True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        return (*lm_head_hip.layer_norm_backward(
            x, weight, ctx.bias_dtype, mean, rstd, dy,
            ctx.needs_input_grad[:3]), None)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) * rstd * weight + bias`` over the last axis of ``x``
    (``[..., C]``), ``rstd = 1 / sqrt(var + eps)``; ``weight`` and ``bias``
    (``[C]``, one dtype, bf16 or fp32 whatever ``x``'s) may be None.  Returns
    ``x``'s shape and dtype."""
    if not _wants_grad(x, weight, bias):
        return lm_head_hip.layer_norm_forward(x, weight, bias, eps, False)[0]
    return _LayerNorm.apply(x, weight, bias, eps)


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor       # [...] fp32, 0 for a token below 0
    entropy: torch.Tensor        # [...] fp32
    top_ids: torch.Tensor | None       # [..., top_k] int64; None with top_k 0
    top_logprobs: torch.Tensor | None  # [..., top_k] fp32


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature):
        lp, ent, ids, top, stats = lm_head_hip.token_logprobs_forward(
            logits, tokens, top_k, temperature, True)
        ctx.save_for_backward(logits, tokens, stats, ent)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(ids, top)
        return lp, ent, ids, top

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp, dent, *_):
        if dlp is None and dent is None:
            return None, None, None, None
        logits, tokens, stats, ent = ctx.saved_tensors
        return lm_head_hip.token_logprobs_backward(
            logits, tokens, ctx.temperature, stats, ent, dlp, dent), \
            None, None, None


def token_logprobs(logits, tokens, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probability of ``tokens`` (``[...]`` int64 or int32) under
    ``softmax(logits / temperature)`` (``[..., V]``), the distribution's
    entropy, and the ``top_k`` (at most 64) likeliest ids with their log
    probabilities, equal ones in the order of their ids.

    A token below 0 (padding, -100) is not scored: its logprob is 0 and it
    has no gradient.  A token of V or more gives NaN.  Logits of -inf are
    masked: probability 0, nothing added to the entropy.  Differentiable in
    ``logits`` through ``logprobs`` and ``entropy``; the alternatives are a
    report and carry no gradient.  A position whose cotangents are zero has a
    zero gradient whatever its logits hold."""
    if not _wants_grad(logits):
        return TokenLogprobs(*lm_head_hip.token_logprobs_forward(
            logits, tokens, top_k, temperature, False)[:4])
    return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top_k,
                                               temperature))


class DistillLoss(NamedTuple):
    loss: torch.Tensor        # fp32 scalar, differentiable in the logits
    row_losses: torch.Tensor  # [...] fp32, each position's, no gradient


class _DistillLoss(torch.autograd.Function):
    """The forward writes the gradient too (the logits are read once); the
    backward hands it on where the loss's own cotangent is 1, which the
    kernel sees on the device, and otherwise has it formed anew."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, weight, temperature):
        loss, rows, d = lm_head_hip.distill_loss_forward(
            logits, ids, teacher, weight, temperature, True)
        ctx.save_for_backward(logits, ids, teacher, weight)
        ctx.temperature, ctx.d = temperature, d
        ctx.mark_non_differentiable(rows)
        ctx.set_materialize_grads(False)
        return loss, rows

    @staticmethod
    @once_differentiable
    def backward(ctx, scale, _):
        if scale is None:
            return None, None, None, None, None
        # a second backward over a retained graph gets a buffer of its own
        d, ctx.d = ctx.d, None
        logits, ids, teacher, weight = ctx.saved_tensors
        return lm_head_hip.distill_loss_backward(
            logits, ids, teacher, weight, ctx.temperature, scale, d), \
            None, None, None, None


def distill_loss(logits, teacher_ids, teacher_logits, weight=None,
                 temperature: float = 1.0) -> DistillLoss:
    """Distillation from a teacher's top logits.

    ``logits`` ``[..., V]`` are the student's; ``teacher_ids`` and
    ``teacher_logits`` ``[..., K]`` (K at most 256, any order) the teacher's
    alternatives, an id below 0 for none.  With ``q = softmax(teacher_logits
    / temperature)`` over the present alternatives and ``p = softmax(logits /
    temperature)`` over the vocabulary, a position's loss is
    ``temperature^2 * KL(q || p)``, and ``loss`` the sum of ``weight`` times
    it (``[...]``; None: the mean over all positions).  An id of V or more
    gives NaN.  A position with weight 0, or with no alternative, has loss
    and gradient 0 whatever its logits hold.

    Where a gradient is wanted the call forms it (for a cotangent of 1 on
    the loss) while it reads the logits; scaling the loss afterwards costs a
    second pass in the backward, scaling ``weight`` nothing.  No gradient
    flows to the teacher or the weight."""
    if not _wants_grad(logits):
        return DistillLoss(*lm_head_hip.distill_loss_forward(
            logits, teacher_ids, teacher_logits, weight, temperature,
            False)[:2])
    return DistillLoss(*_DistillLoss.apply(logits, teacher_ids,
                                           teacher_logits, weight,
                                           temperature))


__all__ = ["DistillLoss", "TokenLogprobs", "distill_loss", "layer_norm",
           "token_logprobs"]
