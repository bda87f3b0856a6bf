/*
 * Operators of a transformer's training step, beside the products and losses of tenmo_hip.h and with its conventions: device
 * pointers, sizes and strides in elements, views over strided storage, one stream, 0 or a negative tenmo_status, the message of a
 * failure in tenmo_hip_last_error().  Of these the reference has a layer norm (tenmo/layernorm.mojo, tenmo/kernels/layernorm.mojo); attention and the loss from the hidden states have no
 * counterpart there.
 *
 * Workspace: an entry that needs scratch memory takes it from the caller (device memory, 256-byte aligned), of at least the bytes that
 * its ..._workspace_bytes function returns for the same sizes.  Nothing is kept in it from one call to the next, and no call
 * allocates or copies to the host: every entry can be captured into a HIP graph (with sync = 0), which then owns the use of the
 * workspace given to it; two calls that may run at the same time need two workspaces.
 *
 * Sizes beyond what a launch holds are refused with TENMO_ERR_UNSUPPORTED: each entry says which.
 *
 * Gradients: with accumulate = 0 they are written, with accumulate != 0 added to what is there.  A NULL gradient is not computed.
 * Results do not depend on scheduling: the same inputs give the same bits.  They share no place with operands or with each other where an entry does not say so.
 *
 * Precision: operands, results and sums are fp32.  Large attention calls, and those of the vocabulary loss on many tokens, multiply on the fp16 matrix units, each fp32 value as a sum of two
 * halves: to 2^-22 of itself, and to 2^-40 of the largest value that has the same scale.  Scales are chosen so that each row of a result is right by itself, however small it is against the others of
 * its call.  Four things remain:
 *   - A probability exp(-t) is off by up to (t + 2) 2^-24 of itself, and by the error of its score or logit, about 2^-22 |q| |k| scale or 2^-22 |h| |w| on the matrix units and 2^-24 of them elsewhere.
 *     The target's p - 1 in the loss's gradient is right to that, not to its own size.
 *   - What a probability is multiplied by does not count in how it is held: attention forward to 2^-28 of the row's largest, backward (and dS) to 2^-35 of the largest that enters the same row of
 *     the result; the loss to 2^-33 of the largest that enters the same row of grad_W, and 2^-40 of 1 for grad_H.  A row that only smaller ones make, because the vectors of the others are zeros,
 *     loses them (output gradients and hidden states of zeros do not count among the others).
 *   - Heads with values that are not finite, with rows of K or V (backward: or Q) whose largest magnitudes lie more than 2^16 apart, rows of zeros aside, or, backward, with scores above 2^16 are
 *     worked on in fp32, value by value: right, but 20 to 140 times as slow as others of their length.
 *   - W of the loss has one scale: each of its values is held to 2^-40 of its largest magnitude at the best, so that the logits of words 2^16 smaller than the largest are as good as fp32 ones and those of
 *     words 2^30 smaller are not.
 * Small calls are in fp32 throughout.
 */
#ifndef TENMO_HIP_TRANSFORMER_H
#define TENMO_HIP_TRANSFORMER_H
#include "tenmo_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- layer norm ---------------------------------------------------------------------------------------------------------- */

/* out[r, :] = (x[r, :] - mean[r]) * rstd[r] * weight + bias over the last axis of X (any strides, rank 1 to 8, N = its last extent >= 1),
 * mean and biased variance of each row, rstd = 1 / sqrt(variance + eps), eps >= 0, N up to 2^27.  weight, bias: N floats or NULL (1 and 0).
 * out: dense, X's shape; it may be X's own place where X is dense.  mean, rstd: one float a row, or NULL (both) when no gradient is wanted. */
int tenmo_hip_layer_norm_forward_f32(const tenmo_view* X, const float* weight, const float* bias, float eps,
                                     float* out, float* mean, float* rstd, int32_t sync);
/* For the upstream gradient dY (dense, X's shape), with xhat = (x - mean) * rstd and g = dY * weight:
 * grad_X = rstd * (g - mean_row(g) - xhat * mean_row(g * xhat)) (dense, X's shape), grad_weight = sum over rows of dY * xhat,
 * grad_bias = sum over rows of dY.  grad_X may be dY's own place, or X's where X is dense, and shares none with them otherwise; grad_weight and grad_bias share none with anything. */
int64_t tenmo_hip_layer_norm_backward_workspace_bytes(int64_t rows, int64_t n);
int tenmo_hip_layer_norm_backward_f32(const tenmo_view* X, const float* weight, const float* mean, const float* rstd, const float* dY,
                                      float* grad_X, float* grad_weight, float* grad_bias, int32_t accumulate,
                                      void* workspace, int64_t workspace_bytes, int32_t sync);

/* ---- attention ------------------------------------------------------------------------------------------------------------ */

/* Q [B, Sq, H, D], K and V [B, Sk, Hk, D] (views with any strides; H a multiple of Hk, query head h reads key head h / (H / Hk);
 * D of 1 to 128; B * H up to 2^20, B * H * Sq up to 2^25, B * Hk * Sk up to 2^27).  out[b, i, h, :] = sum over the allowed keys j of softmax_j(scale * q_i . k_j) * v_j, dense [B, Sq, H, D].
 * Key j is allowed for query i of sequence b when j < key_lengths[b] (NULL: Sk; taken as 0 below 0 and as Sk above Sk) and, if causal != 0,
 * j <= i + query_starts[b] (the position of the first query; NULL: Sk - Sq, the queries are the last positions).  Both are device arrays
 * of B ints.  Keys that are not allowed are not used, whatever they hold; a query without keys gets zeros.
 * lse: NULL, or dense [B, H, Sq]: log of the sum of exp(scale * q_i . k_j) over the allowed keys (-inf without keys), for the backward call.
 * The size of the workspace depends on the device: the function needs tenmo_hip_init, and returns a negative status without. */
int64_t tenmo_hip_attention_forward_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim);
int tenmo_hip_attention_forward_f32(const tenmo_view* Q, const tenmo_view* K, const tenmo_view* V, float scale, int32_t causal,
                                    const int32_t* key_lengths, const int32_t* query_starts, float* out, float* lse,
                                    void* workspace, int64_t workspace_bytes, int32_t sync);
/* Gradients for the upstream gradient dOut (dense [B, Sq, H, D]); out and lse as the forward call with the same arguments left them.  The
 * probabilities are computed again.  grad_Q, grad_K, grad_V: views of the shapes of Q, K, V with strides of their own (no two elements
 * of the three at one place), written through; grad_K and grad_V sum over the query heads that share a key head.
 * Where heads are shared, B * H * Sk up to 2^28. */
int64_t tenmo_hip_attention_backward_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim);
int tenmo_hip_attention_backward_f32(const tenmo_view* Q, const tenmo_view* K, const tenmo_view* V, float scale, int32_t causal,
                                     const int32_t* key_lengths, const int32_t* query_starts, const float* out, const float* lse,
                                     const float* dOut, const tenmo_view* grad_Q, const tenmo_view* grad_K, const tenmo_view* grad_V,
                                     int32_t accumulate, void* workspace, int64_t workspace_bytes, int32_t sync);

/* ---- cross-entropy over a vocabulary, from the hidden states ---------------------------------------------------------------- */

/* tenmo_hip_cross_entropy_forward_f32 of the logits H . W + bias without writing them: H [M, D] and W [D, V] are views of any strides (a weight
 * tied to an embedding [V, D] is its transposed view), bias V floats or NULL; target, ignore_index, label_smoothing, per_sample_loss [M],
 * loss_sum [1] and valid_count [1] as there (a target outside 0..V-1 that is not ignore_index gives NaN).  lse [M]: log of the sum of the
 * exponentials of each row of logits.  M and V up to 2^22, D up to 2^20, each product of two of them up to 2^38.  A row of H or a word of W that is not finite
 * makes the results that it enters not finite; the hidden state of an ignored token enters its own lse alone. */
int64_t tenmo_hip_vocabulary_loss_forward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocabulary);
int tenmo_hip_vocabulary_loss_forward_f32(const tenmo_view* H, const tenmo_view* W, const float* bias, const void* target,
                                          int32_t target_is_int64, int64_t ignore_index, float label_smoothing,
                                          float* per_sample_loss, float* lse, float* loss_sum, int32_t* valid_count,
                                          void* workspace, int64_t workspace_bytes, int32_t sync);
/* With G the gradient of tenmo_hip_cross_entropy_backward_f32 (reduction 0 none: upstream [M], 1 sum and 2 mean: upstream [1]; valid_count is the
 * DEVICE int that the forward call wrote, read for the mean alone): grad_H = G . W^T (dense [M, D]), grad_W = H^T . G (a view of W's shape with
 * strides of its own, no two elements at one place), grad_bias = sum over rows of G.  lse as the forward call left it.  The logits are computed again, a piece of the
 * vocabulary at a time. */
int64_t tenmo_hip_vocabulary_loss_backward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocabulary);
int tenmo_hip_vocabulary_loss_backward_f32(const tenmo_view* H, const tenmo_view* W, const float* bias, const void* target,
                                           int32_t target_is_int64, int64_t ignore_index, float label_smoothing, const float* lse,
                                           const float* upstream, int32_t reduction, const int32_t* valid_count,
                                           float* grad_H, const tenmo_view* grad_W, float* grad_bias, int32_t accumulate,
                                           void* workspace, int64_t workspace_bytes, int32_t sync);

#ifdef __cplusplus
}
#endif
#endif /* TENMO_HIP_TRANSFORMER_H */
