/*
 * mxs_head.h -- C ABI of the output-head operators of the B200 (sm_100a) token
 * sampler library: what the head is scored and trained with (the softmax cross
 * entropy over the vocabulary, from hidden states, with its gradients) and what
 * it is served with in 8 bits (quantiser, block-scaled matrix product, and the
 * sampler on its logits).
 *
 * The reference computes the head's logits of a step and samples them
 * (src/api/minxfmr.cpp:1918-2036, :2091-2171); it has no loss, no gradient and no
 * 8-bit floating type, so these entry points have no counterpart there.
 *
 * Conventions as mxs_sampler.h: 0 on success, a negative code on error, nothing
 * throws; device pointers are the caller's; calls are asynchronous on `stream`
 * and read no host memory after they return. No call allocates device memory:
 * scratch is the caller's workspace (256-byte aligned, at least as large as the
 * matching *_workspace_size says, any contents), so calls on different streams
 * run side by side when each has its own, and a call can be captured in a CUDA
 * graph. Outputs do not depend on timing: no floating-point atomics.
 * A bounded device wait that gives up is reported by mxs_get_status
 * (MXS_ROW_TIMEOUT); the call's outputs are then invalid.
 */
#ifndef MXS_HEAD_H
#define MXS_HEAD_H

#include "mxs_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of operands and outputs. */
#define MXS_BF16 0
#define MXS_F16 1
#define MXS_F32 2

/*
 * Softmax cross entropy of rows against a vocabulary, from hidden states; the
 * logits are never stored. With x_v = <hidden_r, weight_v> / temperature:
 *   loss_r = -log softmax(x)_t = log(1 + sum_{v != t} exp(x_v - x_t)),  t = target of row r
 *   lse_r  = log sum_v exp(x_v)
 * (-loss_r is the log-probability of token t under the distribution that
 * mxs_sample_from_hidden draws from at top_k = vocab and this temperature.)
 *   d_hidden  rows x d_model of `dtype` (MXS_BF16 or MXS_F16), row r at d_hidden + r*ld_hidden elements
 *   d_weight  vocab x d_model of `dtype`, row v at d_weight + v*ld_weight elements
 *   d_targets rows integers of target_bytes (4 or 8) bytes. A row whose target is
 *             outside [0, vocab) is left out: loss and lse are 0, and its hidden
 *             state (it may hold NaN) reaches no output. Above 128 rows it is not
 *             read either and costs no products.
 *   d_loss, d_lse  rows floats; either may be NULL
 * Products are accumulated in fp32, rounded towards zero within runs of 128 (up to
 * 128 rows) or 512 and to nearest between them; maxima and sums of the softmax are
 * fp32. Limits: vocab, rows, d_model < 2^31 - 1024; temperature > 0.
 */
MXS_API int mxs_ce_from_hidden(const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight,
                               int dtype, int64_t rows, int64_t d_model, int64_t vocab, const void* d_targets,
                               int target_bytes, double temperature, float* d_loss, float* d_lse, void* d_workspace,
                               size_t workspace_bytes, void* stream);

/*
 * Gradients of sum_r grad_loss_r * loss_r, from the lse of mxs_ce_from_hidden on
 * the same operands (d_lse is read for rows with a target in range only):
 *   P[r][v] = softmax(x_r)_v - (v == t_r)            (rows left out: 0)
 *   grad_hidden_r = grad_loss_r / temperature * sum_v P[r][v] weight_v
 *   grad_weight_v = 1 / temperature * sum_r grad_loss_r P[r][v] hidden_r
 * Both are written whole (rows left out get a zero gradient); either may be NULL
 * and is then not computed. The logits are computed again, a piece of the
 * vocabulary at a time; a piece of grad_loss_r P[r][v] / max |grad_loss| is held in
 * `dtype` (entries below 2^-28 (MXS_F16) or 2^-126 (MXS_BF16) lose precision),
 * what that rounding leaves out of a row's target entry is kept in fp32, sums are
 * fp32, and the gradients are rounded to `dtype` once. At most 2^24 rows a call.
 */
MXS_API int mxs_ce_from_hidden_backward(const void* d_hidden, int64_t ld_hidden, const void* d_weight,
                                        int64_t ld_weight, int dtype, int64_t rows, int64_t d_model, int64_t vocab,
                                        const void* d_targets, int target_bytes, double temperature,
                                        const float* d_lse, const float* d_grad_loss, void* d_grad_hidden,
                                        int64_t ld_grad_hidden, void* d_grad_weight, int64_t ld_grad_weight,
                                        void* d_workspace, size_t workspace_bytes, void* stream);

/*
 * Bytes of workspace the two calls above need (backward: 0 or 1). d_weight is
 * not read; its alignment and ld_weight count: a weight whose rows do not start
 * on 16-byte boundaries is copied into aligned rows first, which takes room for
 * the copy and another pass over it.
 */
MXS_API int mxs_ce_workspace_size(const void* d_weight, int64_t ld_weight, int64_t rows, int64_t d_model,
                                  int64_t vocab, int backward, size_t* bytes);

/*
 * 8-bit floats (4 exponent bits, 3 mantissa bits, largest value 448) with one
 * fp32 scale for each block of block_rows x 128 elements (block_rows: 1 for
 * activations, 128 for weights; blocks at the right and lower edges are cut):
 *   scale = max(largest finite magnitude of the block / 448, 2^-126), 1 for a block of zeros
 *   q     = round to nearest even (x / scale), saturated to +-448; NaN stays NaN
 *   d_x      rows x cols of `dtype` (MXS_BF16, MXS_F16 or MXS_F32), leading dimension ld_x
 *   d_q      rows x cols bytes, leading dimension ld_q (16-byte aligned rows make mxs_matmul_fp8 fastest)
 *   d_scale  ceil(rows / block_rows) x ceil(cols / 128) floats, contiguous
 */
MXS_API int mxs_quantize_fp8(const void* d_x, int64_t ld_x, int dtype, int64_t rows, int64_t cols, int block_rows,
                             void* d_q, int64_t ld_q, float* d_scale, void* stream);

/*
 * out[r][j] = sum_k a_scale[r][k/128] * b_scale[j/128][k/128] * a[r][k] * b[j][k]:
 * the product of a rows x k and an n x k matrix of 8-bit floats with a scale
 * for each 1 x 128 block of a and each 128 x 128 block of b, as
 * mxs_quantize_fp8 makes them. Each block of 128 products is summed in fp32 and
 * joined under its scales in fp32, whose product is formed first (it keeps its 24
 * bits between 2^-126 and 2^128); out (MXS_F32, MXS_BF16 or MXS_F16; leading
 * dimension ld_out) is rounded once. Limits: rows, n, k < 2^31 - 1024.
 */
MXS_API int mxs_matmul_fp8(const void* d_a, int64_t ld_a, const float* d_a_scale, const void* d_b, int64_t ld_b,
                           const float* d_b_scale, int64_t rows, int64_t n, int64_t k, void* d_out, int64_t ld_out,
                           int out_dtype, void* d_workspace, size_t workspace_bytes, void* stream);

/* Bytes of workspace mxs_matmul_fp8 needs (the pointers are not read; operands whose rows do not
 * start on 16-byte boundaries are copied into aligned rows first). */
MXS_API int mxs_matmul_fp8_workspace_size(const void* d_a, int64_t ld_a, const void* d_b, int64_t ld_b, int64_t rows,
                                          int64_t n, int64_t k, size_t* bytes);

/*
 * mxs_sample_from_hidden with the head's weight in 8 bits: the hidden states
 * (`dtype` MXS_BF16 or MXS_F16) are quantised with a scale for each row's 128
 * columns, multiplied into fp32 logits, and sampled where they land
 * (mxs_sample_topk_ex). The workspace holds the quantised rows, the logits
 * unless d_logits_out is given, and the sampler's own workspace (which the call
 * clears); its size comes from the query below.
 */
MXS_API int mxs_sample_from_hidden_fp8(const void* d_hidden, int64_t ld_hidden, int dtype, const void* d_weight_q,
                                       int64_t ld_weight, const float* d_weight_scale, int64_t rows, int64_t d_model,
                                       int64_t vocab, double temperature, int top_k, double top_p, double min_p,
                                       const double* d_u, int32_t* d_next, int32_t* d_topk_idx, double* d_topk_prob,
                                       float* d_logits_out, int64_t ld_logits, void* d_workspace,
                                       size_t workspace_bytes, void* stream);

/* Bytes of workspace mxs_sample_from_hidden_fp8 needs. */
MXS_API int mxs_sample_from_hidden_fp8_workspace_size(const void* d_weight_q, int64_t ld_weight, int64_t rows,
                                                      int64_t d_model, int64_t vocab, int top_k, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* MXS_HEAD_H */
