"""Operators around a language model's head.

The end of the model and what is made of its logits:

* ``layer_norm``: the norm before the head, as before each block's mixes;
* ``token_logprobs``: log probabilities of given tokens, entropy and the top
  alternatives, for scoring, for a decode step's report and, being
  differentiable, for training on them;
* ``distill_loss``: the distillation loss from a teacher's top logits, whose
  gradient is formed in the same pass over the logits;
* ``verify_drafts``: which of a sequence's drafted tokens the model takes, and
  the token behind them, from given random numbers.

The head's product between the first and the others is a plain GEMM and
stays the caller's (``x @ head.T``).  Each is one or two HIP kernels
(``kernels/lm_head_hip.py``); tensors are on the GPU, activations and logits
bf16 or fp32, and every sum is held in fp32 or more.  Gradients are first
order and reverse mode: a second derivative or a forward-mode tangent raises.
``examples/distill_and_score.py`` runs the first three together.
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


class VerifiedDrafts(NamedTuple):
    tokens: torch.Tensor    # [B, K + 1] int64: the drafts taken, one more, -1
    accepted: torch.Tensor  # [B] int64, how many drafts were taken
    chances: torch.Tensor   # [B, K] fp32, each draft's chance to be taken


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


def verify_drafts(logits, draft_tokens, draft_logits=None,
                  accept_uniforms=None, sample_uniforms=None,
                  draft_lengths=None,
                  temperature: float = 1.0) -> VerifiedDrafts:
    """Verify drafted tokens (``draft_tokens`` ``[B, K]`` int64 or int32, K at
    most 64) against a model's ``logits`` ``[B, K + 1, V]``, row i those that
    follow the first i drafts, so that what is emitted is distributed as the
    model's own samples are.

    With ``p = softmax(logits / temperature)`` and ``q = softmax(draft_logits
    / temperature)`` (``[B, K, V]``, the dtype of ``logits``; None where the
    drafts are certain, found by lookup, not drawn), draft x of a position is
    taken while ``accept_uniforms * q(x) < p(x)``; behind the ``accepted``
    ones a token is drawn from ``max(p - q, 0)`` of the first position not
    taken (from its ``p`` where nothing is left of that, p being q), or from
    the last row's ``p`` where all were, by ``sample_uniforms`` along the
    running sum over the vocabulary.  A draft outside the vocabulary is never
    taken.  ``accept_uniforms`` ``[B,
    K]`` and ``sample_uniforms`` ``[B]`` are fp32, from 0 to below 1; they are
    compared in float64.  ``draft_lengths`` ``[B]`` (int64 or int32) gives
    sequences with fewer drafts than K; rows past them are not read.

    ``temperature=0.0`` is greedy: a draft is taken where it is the likeliest
    token (the lowest id of equal ones), which is also the one emitted behind
    them; ``draft_logits`` and the random numbers are not looked at.

    ``tokens`` holds the drafts taken, the token drawn, then -1.  ``accepted +
    1`` is the number of tokens by which the sequence goes on: the
    ``lengths`` of ``gated_delta_step``.  A token is -1 where its row has no
    distribution (it, or the draft's, holds NaN or +inf, or nothing above
    -inf); chances of such rows are NaN.

    There is no gradient: logits that require one are refused where gradients
    are enabled, as are forward-mode tangents."""
    return VerifiedDrafts(*load_binding().verify_drafts(
        logits, draft_tokens, draft_logits, accept_uniforms, sample_uniforms,
        draft_lengths, temperature))


__all__ = ["DistillLoss", "TokenLogprobs", "VerifiedDrafts", "distill_loss",
           "layer_norm", "token_logprobs", "verify_drafts"]
