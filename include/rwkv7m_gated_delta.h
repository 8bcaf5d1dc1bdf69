/*
 * rwkv7m_gated_delta.h -- C ABI of the gated delta rule in librwkv7m_wkv.so:
 * the recurrence of a linear-attention head whose state decays by one factor
 * a token and writes along its key what the state does not say there already,
 *
 *   S_t = e^{g_t} S_{t-1} (I - beta_t k_t k_t^T) + beta_t v_t k_t^T,
 *   o_t = scale S_t q_t,
 *
 * S [Dv][Dk], rows of values as in rwkv7m_wkv.h (wkv7 with decay e^g in every
 * column, neg_kk = -k, kka = e^g beta k and beta k for k is the same
 * recurrence).  Status codes, dtype codes and rwkv7m_last_error() are those of
 * rwkv7m_wkv.h.
 *
 * q and k have Hk heads of Dk, v, o and the gates g and beta Hv, a multiple of
 * Hk: value head h reads key head h / (Hv / Hk).  8 <= Dk <= 128 and 8 <= Dv
 * <= 256, multiples of 8.  Vectors are bf16 or fp32, one dtype; g and beta
 * each bf16 or fp32; states fp32.  Vectors and gates are read where they lie:
 * each has a stride (in elements, >= 0) for batch, token and head; a vector's
 * places are adjacent, and it starts at a multiple of 16 bytes (v and the
 * outputs of the step: 8).  Outputs and gradients are contiguous [B][T][H][D]
 * (gates [B][T][Hv]); an output shares no byte with an input, the step's state
 * excepted.
 *
 * Keys are taken as they come: the recurrence contracts where beta |k|^2 <= 2
 * and g <= 0, and grows where it does not.  g of -inf clears the state.  A
 * number that is not finite makes what it reaches NaN, and may make the rest of
 * its chunk of 64 tokens NaN, tokens before it among them.
 *
 * Sums and states are fp32, products bf16 matrix instructions over sums of
 * three bf16 planes, which hold what fp32 does: results are off as with fp32
 * products, some 2e-7 to 5e-7 of their norm (dg, a small sum of large terms, up
 * to 2e-6; all up to 3e-6 where beta |k|^2 nears 2 and keys hardly differ),
 * before they are rounded to their own type.  Calls only
 * enqueue work on `stream`, never allocate and never synchronise, so they may
 * be captured in a HIP graph.  Results do not depend on the order in which
 * workgroups run, nor a sequence's on the others in its batch.
 */
#ifndef RWKV7M_GATED_DELTA_H
#define RWKV7M_GATED_DELTA_H

#include <stdint.h>

#include "rwkv7m_wkv.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int dtype, g_dtype, beta_dtype;
    int64_t B, T, Hk, Hv, Dk, Dv;
    const void *q, *k, *v, *g, *beta;
    /* batch, token, head */
    int64_t q_stride[3], k_stride[3], v_stride[3], g_stride[3], beta_stride[3];
    double scale;
} rwkv7m_gated_delta_inputs;

/* Bytes of device workspace of a call (-1 for invalid sizes): 16-byte
 * aligned, free again once the call's work is done. */
int64_t rwkv7m_gated_delta_workspace_bytes(const rwkv7m_gated_delta_inputs *in,
                                           int backward);

/* Floats that a forward keeps for the backward (-1 for invalid sizes). */
int64_t rwkv7m_gated_delta_saved_floats(const rwkv7m_gated_delta_inputs *in);

/* o [B][T][Hv][Dv]; initial_state [B][Hv][Dv][Dk] or NULL (zeros); final_state
 * the same or NULL (not wanted); saved NULL, or what the backward takes (the
 * workspace is then not needed). */
int rwkv7m_gated_delta_rule(const rwkv7m_gated_delta_inputs *in,
                            const float *initial_state, void *o,
                            float *final_state, float *saved, void *workspace,
                            int64_t workspace_bytes, void *stream);

/* Gradients for the cotangents d_o (with strides as the vectors') and
 * d_final_state (NULL: zeros): dq, dk, dv of the vectors' dtype, dg and dbeta
 * of their gate's, d_initial_state fp32 or NULL (not wanted).  dq and dk are
 * summed over the value heads that share a key head. */
int rwkv7m_gated_delta_rule_backward(
    const rwkv7m_gated_delta_inputs *in, const void *d_o,
    const int64_t *d_o_stride, const float *d_final_state, const float *saved,
    void *dq, void *dk, void *dv, void *dg, void *dbeta,
    float *d_initial_state, void *workspace, int64_t workspace_bytes,
    void *stream);

/* The recurrence for short blocks of T tokens (decode) on a pool of states
 * [pool][Hv][Dv][Dk], updated in place, or only read with update = 0.  Row b
 * goes on from state slots[b] (NULL: b) over its first lengths[b] tokens
 * (NULL, or more than T: T); o is 0 behind them.  A slot below 0 is padding:
 * o is 0.  A slot of `pool` or more, or one that an earlier row of the same
 * call updates, gives NaN in o and leaves the state to the earlier row. */
int rwkv7m_gated_delta_step(const rwkv7m_gated_delta_inputs *in, int64_t pool,
                            float *state, const int64_t *slots,
                            const int64_t *lengths, int update, void *o,
                            void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV7M_GATED_DELTA_H */
