"""The gated delta rule: the recurrence of a linear-attention head whose state
``S`` (``[Dv, Dk]``, rows of values as in ``wkv7``) decays by one factor a
token and writes along its key what it does not say there already:

    S_t = exp(g_t) S_{t-1} (I - beta_t k_t k_t^T) + beta_t v_t k_t^T
    o_t = scale * S_t q_t

* ``gated_delta_rule``: whole sequences, in chunks, differentiable;
* ``gated_delta_step``: a token, or a short block of drafted ones, on a pool of
  states updated in place.

It is ``wkv7`` with one decay a head (``neg_kk = -k``, ``kka = exp(g) beta k``,
``beta k`` for ``k``); what it adds are value heads that share key heads, head
sizes that differ between keys and values, and a fraction of the bytes, since
the gates are one number a head.

Vectors are batch-major, ``q`` and ``k`` ``[B, T, Hk, Dk]``, ``v`` ``[B, T, Hv,
Dv]``, bf16 or fp32, one dtype; the gates ``g`` and ``beta`` ``[B, T, Hv]``,
each bf16 or fp32; value head h reads key head ``h // (Hv // Hk)``; Dk is a
multiple of 8 up to 128, Dv one up to 256.  They are read where they lie as
long as the last axis of a vector is dense and its rows start at multiples of
16 bytes (views of one fused projection do); others are copied first.  Keys
are taken as they come: normalise them (the recurrence contracts where ``beta
|k|^2 <= 2`` and ``g <= 0``).  Padding tokens with ``beta`` and ``g`` 0 leave the
state as it is, if their vectors are finite.  States are fp32.  Kernels run on the current stream
(``csrc/gdr_*.hip``, C ABI in ``include/rwkv7m_gated_delta.h``); there is no
CPU fallback.
"""

from __future__ import annotations

from .kernels.lm_head_hip import load_binding


def gated_delta_rule(q, k, v, g, beta, initial_state=None,
                     scale: float | None = None):
    """``(o, final_state)``: ``o`` ``[B, T, Hv, Dv]`` of the vectors' dtype and
    the fp32 state ``[B, Hv, Dv, Dk]`` after the last token, from
    ``initial_state`` (None: zeros).  ``scale`` is ``Dk ** -0.5`` by default.

    Differentiable, first order and reverse mode, in the five inputs and the
    initial state, through both outputs; a second derivative or a
    forward-mode tangent raises.  While it runs the call takes 38 KB a value
    head and chunk of 64 tokens, the chunk's matrices.  For the backward it
    keeps these, and a value head and chunk the fp32 state before it and its
    tokens' writes, ``4 Dv (Dk + 64)`` bytes with Dk rounded up to 64 or 128
    and Dv to a multiple of 32; the backward takes the latter as much again
    while it runs, and where value heads share key heads ``8 Hv Dk`` bytes a
    token.

    A number that is not finite makes what it reaches NaN, and may make the
    rest of its chunk of 64 tokens in its head NaN, tokens before it among
    them.

    To capture a backward pass in a graph, use leaves that no live eager graph
    holds (detached clones do): the engine would wait across streams, which a
    capture does not survive."""
    return load_binding().gated_delta_rule(q, k, v, g, beta, initial_state,
                                           scale)


def gated_delta_step(q, k, v, g, beta, state, lengths=None, slots=None,
                     scale: float | None = None, update_state: bool = True):
    """``o`` ``[B, T, Hv, Dv]`` of a short block of tokens (T = 1 for plain
    decoding), going on from ``state`` ``[pool, Hv, Dv, Dk]``, contiguous fp32,
    which is updated in place.

    ``slots`` ``[B]`` (int64 or int32) names each row's state in the pool
    (None: row b's is b); one below 0 is padding, whose ``o`` is 0.
    ``lengths`` ``[B]`` gives rows with fewer tokens than T; ``o`` is 0 behind
    them.  A slot past the pool, or one that an earlier row of the call
    updates, gives NaN in ``o`` and leaves the state to the earlier row.

    ``update_state=False`` reads a block ahead and leaves the states as they
    are: verify it (``verify_drafts``), then call again with ``lengths =
    accepted + 1``.  There is no gradient."""
    return load_binding().gated_delta_step(q, k, v, g, beta, state, lengths,
                                           slots, scale, update_state)


__all__ = ["gated_delta_rule", "gated_delta_step"]
