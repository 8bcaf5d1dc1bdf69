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
order and reverse mode: a second derivative or a forward-mode tangent raises.
``examples/distill_and_score.py`` runs the three together.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .kernels.lm_head_hip import load_binding


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor       # [...] fp32, 0 for a token below 0
    entropy: torch.Tensor        # [...] fp32
    top_ids: torch.Tensor | None       # [..., top_k] int64; None with top_k 0
    top_logprobs: torch.Tensor | None  # [..., top_k] fp32


class DistillLoss(NamedTuple):
    loss: torch.Tensor        # fp32 scalar, differentiable in the logits
    row_losses: torch.Tensor  # [...] fp32, each position's, no gradient


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) * rstd * weight + bias`` over the last axis of ``x``
    (``[..., C]``), ``rstd = 1 / sqrt(var + eps)``; ``weight`` and ``bias``
    (``[C]``, one dtype, bf16 or fp32 whatever ``x``'s) may be None.  Returns
    ``x``'s shape and dtype."""
    return load_binding().layer_norm(x, weight, bias, eps)


def token_logprobs(logits, tokens, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probability of ``tokens`` (``[...]`` int64 or int32) under
    ``softmax(logits / temperature)`` (``[..., V]``; temperatures from 1e-30 to
    1e30), the distribution's entropy, and the ``top_k`` (at most 64) likeliest ids with their log
    probabilities, equal ones in the order of their ids.

    A token below 0 (padding, -100) is not scored: its logprob is 0, whatever
    its position's logits hold, and it has no gradient.  A token of V or more
    gives NaN.  Logits of -inf are masked: probability 0, nothing added to the
    entropy.  Differentiable in ``logits`` through ``logprobs`` and
    ``entropy``; the alternatives are a report and carry no gradient.  A
    position whose cotangents are zero has a zero gradient whatever its logits
    hold."""
    return TokenLogprobs(*load_binding().token_logprobs(logits, tokens, top_k,
                                                        temperature))


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
    second pass in the backward, scaling ``weight`` nothing.  Until the
    backward the gradient is held beside the saved logits, out of reach of
    saved-tensor hooks.  No gradient flows to the teacher or the weight."""
    return DistillLoss(*load_binding().distill_loss(
        logits, teacher_ids, teacher_logits, weight, temperature))


__all__ = ["DistillLoss", "TokenLogprobs", "distill_loss", "layer_norm",
           "token_logprobs"]
