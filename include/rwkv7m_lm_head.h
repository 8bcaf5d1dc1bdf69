/*
 * rwkv7m_lm_head.h -- C ABI of the operators around a language model's head
 * in librwkv7m_wkv.so: the layer norm before it (and before each block's
 * mixes), the log probabilities, entropy and top alternatives read from its
 * logits, and the distillation loss from a teacher's top logits.  Status
 * codes, dtype codes and rwkv7m_last_error() are those of rwkv7m_wkv.h.  The
 * head's product itself is a plain GEMM left to the caller's library.
 *
 * Rows.  x and logits are read where they lie: row r of rows = outer * inner
 * starts at (r / inner) * outer_stride + (r % inner) * inner_stride elements,
 * its elements are adjacent, and it needs no more than its element type's
 * alignment.  (logits[:, :-1] of a [B, T, V] tensor is outer = B, inner =
 * T - 1, outer_stride = T * V, inner_stride = V.)  Every other array is
 * contiguous.  Statistics and sums are fp32 or wider; bf16 results are
 * rounded once, to nearest even.  Strides are >= 0 elements; an output shares
 * no byte with an input.  Calls only enqueue work on `stream`, never allocate
 * and never synchronise, so they may be captured in a HIP graph.  Results do
 * not depend on the order in which workgroups run, nor a row's on how many
 * others there are.  A row of logits is summed in an order that goes by its
 * address modulo 16 bytes and, up to 8192 bytes, by whether more than 40
 * alternatives are asked for or a teacher gives more than 64: between those
 * its values agree to rounding, not to the last bit.  (Rows of a batch whose
 * length is no multiple of 16 bytes lie at different such addresses.)
 */
#ifndef RWKV7M_LM_HEAD_H
#define RWKV7M_LM_HEAD_H

#include <stdint.h>

#include "rwkv7m_wkv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest number of alternatives that rwkv7m_token_logprobs returns, and
 * that a teacher gives rwkv7m_distill_loss. */
#define RWKV7M_MAX_TOP_K 64
#define RWKV7M_MAX_TEACHER_K 256

/* y = (x - mean) * rstd * weight + bias over the C elements of each row, with
 * rstd = 1 / sqrt(mean((x - mean)^2) + eps).  x and y of `dtype`; weight and
 * bias (C elements each of `param_dtype`) may be NULL (1 and 0).  mean and
 * rstd [rows] fp32 are what the backward takes; NULL where there is none.  A
 * row's sum and the sum of its squared deviations have to fit fp32. */
int rwkv7m_layer_norm(int dtype, int param_dtype, int64_t outer, int64_t inner,
                      int64_t C, int64_t outer_stride, int64_t inner_stride,
                      const void *x, const void *weight, const void *bias,
                      double eps, void *y, float *mean, float *rstd,
                      void *stream);

/* Floats of device workspace the backward needs (-1 for invalid sizes). */
int64_t rwkv7m_layer_norm_workspace_floats(int64_t rows, int64_t C);

/* With g = dy * weight and xh = (x - mean) * rstd:
 *   dx = rstd * (g - mean(g) - xh * mean(g * xh)),
 *   dweight = sum over rows of dy * xh,  dbias = sum over rows of dy.
 * dy and dx [rows][C] of `dtype`; dweight and dbias of `param_dtype`.  Each
 * of the three results may be NULL (not wanted). */
int rwkv7m_layer_norm_backward(int dtype, int param_dtype, int64_t outer,
                               int64_t inner, int64_t C, int64_t outer_stride,
                               int64_t inner_stride, const void *x,
                               const void *weight, const float *mean,
                               const float *rstd, const void *dy, void *dx,
                               void *dweight, void *dbias, float *workspace,
                               int64_t workspace_floats, void *stream);

/* Over the V logits x of each row, with z = x / temperature and p =
 * softmax(z):
 *   logprobs[r] = log p[tokens[r]];  entropy[r] = -sum p log p;
 *   top_ids[r], top_logprobs[r]: the top_k largest logits, equal ones in the
 *   order of their ids, and their log p ([rows][top_k]; NULL with top_k 0).
 * tokens int64: one below 0 is not scored (logprob 0 whatever its row holds),
 * one >= V gives NaN.  An element of -inf has p = 0 and adds nothing; in a row
 * of nothing else every log p is -inf and the entropy 0.  A row that holds NaN
 * or +inf has NaN in place of the others; NaN ranks above +inf.  0 <= top_k <=
 * min(V, RWKV7M_MAX_TOP_K), 1e-30 <= temperature <= 1e30.  `stats` [rows][2]
 * is what the backward takes (NULL where there is none). */
int rwkv7m_token_logprobs(int dtype, int64_t outer, int64_t inner, int64_t V,
                          int64_t outer_stride, int64_t inner_stride,
                          const void *logits, const int64_t *tokens,
                          int64_t top_k, double temperature, float *logprobs,
                          float *entropy, int64_t *top_ids,
                          float *top_logprobs, float *stats, void *stream);

/* dlogits[r][j] = (1 / temperature) * (d_logprobs[r] * ((j == tokens[r]) -
 * p_j) - d_entropy[r] * p_j * (log p_j + entropy[r])), [rows][V] of `dtype`.
 * d_logprobs and d_entropy [rows] fp32, either may be NULL (zero).  A token
 * below 0 takes no part in its row's logprob.  A row whose cotangents are all
 * zero has a zero gradient and its logits are not read. */
int rwkv7m_token_logprobs_backward(
    int dtype, int64_t outer, int64_t inner, int64_t V, int64_t outer_stride,
    int64_t inner_stride, const void *logits, const int64_t *tokens,
    double temperature, const float *stats, const float *entropy,
    const float *d_logprobs, const float *d_entropy, void *dlogits,
    void *stream);

/* Distillation from a teacher's top K logits (K <= RWKV7M_MAX_TEACHER_K).
 * With q = softmax(teacher_logits / T) over the row's present alternatives
 * (id >= 0) and p = softmax(logits / T) over V:
 *   row_losses[r] = T^2 * sum_k q_k (log q_k - log p[id_k]),
 *   loss[0] = sum_r weight[r] * row_losses[r],
 *   dlogits[r][j] = weight[r] * T * (p_j - sum over k with id_k = j of q_k).
 * teacher_ids int64 and teacher_logits (of `teacher_dtype`) [rows][K]; an id
 * >= V gives NaN; an alternative of -inf has q = 0 and adds nothing.  weight
 * [rows] fp32, or NULL: 1 / rows each.  A row with weight 0, or without an
 * alternative above -inf, has loss and gradient 0 whatever its logits hold.
 * In the other rows NaN or +inf among the logits makes loss and gradient NaN,
 * among the present teacher's the loss and the gradient at its ids; a logit of
 * -inf has p = 0, and the loss is +inf where q > 0 there (the gradient stays
 * finite: -weight T q).
 * row_losses [rows] fp32, off by fp32's rounding of T^2 max(1, |log p|);
 * dlogits [rows][V] of `dtype`, or NULL: the losses alone.  1e-30 <=
 * temperature <= 1e30. */
int rwkv7m_distill_loss(int dtype, int teacher_dtype, int64_t outer,
                        int64_t inner, int64_t V, int64_t outer_stride,
                        int64_t inner_stride, int64_t K, const void *logits,
                        const int64_t *teacher_ids, const void *teacher_logits,
                        const float *weight, double temperature, float *loss,
                        float *row_losses, void *dlogits, void *stream);

/* The gradient of scale[0] * loss, `scale` one fp32 on the device.  With
 * holds_unit != 0 dlogits already holds rwkv7m_distill_loss's, and nothing is
 * done where scale[0] is 1 (decided on the device, without a
 * synchronisation); otherwise the gradient is computed anew from the logits,
 * so that it is rounded once. */
int rwkv7m_distill_loss_backward(
    int dtype, int teacher_dtype, int64_t outer, int64_t inner, int64_t V,
    int64_t outer_stride, int64_t inner_stride, int64_t K, const void *logits,
    const int64_t *teacher_ids, const void *teacher_logits,
    const float *weight, double temperature, const float *scale,
    int holds_unit, void *dlogits, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV7M_LM_HEAD_H */
