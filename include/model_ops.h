/*
 * slideformer_amd -- C-ABI of the operators at a language model's two ends on
 * MI355X (gfx950): embedding lookup and its gradient, the root-mean-square norm
 * with the residual's addition and its gradient, and softmax cross entropy over
 * a vocabulary matrix with its gradients.
 *
 * Plain pointers and sizes only; no torch types.  The caller owns every buffer
 * and every workspace; the library allocates nothing and keeps no state.
 * Matrices are row-major with contiguous rows; a *_stride is the distance of
 * two rows in elements.
 *
 * Return codes are those of layer_adam.h: 0 on success; LA_EINVAL for a null or
 * misaligned pointer, a bad size or a workspace that is too small; LA_EDTYPE
 * for element types an operator does not take; LA_EFAULT for a pointer that is
 * not device memory; a positive hipError_t when a HIP call fails.  No C++
 * exception leaves the library.  All checks come before the first launch, and
 * every call is asynchronous on the stream passed in.
 */
#ifndef SLIDEFORMER_AMD_MODEL_OPS_H
#define SLIDEFORMER_AMD_MODEL_OPS_H

#include "layer_adam.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LA_OPS_ABI_VERSION 1

/* element types of token ids, and of 8-bit outputs */
#define LA_I32 16
#define LA_I64 17
#define LA_I8 18
#define LA_F8E4M3 19

int la_ops_abi_version(void);

/*
 * out[i, :] = scale * weight[tokens[i], :], rounded once.  A token outside
 * [0, vocab) gives a row of NaN.  dtype: LA_F32, LA_BF16 or LA_F16.
 */
int la_embedding(int token_dtype, const void* tokens, uint64_t n, int dtype, const void* weight, uint64_t vocab,
                 uint64_t hidden, uint64_t weight_stride, float scale, void* out, uint64_t out_stride,
                 la_stream_t stream);

/*
 * grad_weight[t, :] = (accumulate ? grad_weight[t, :] : 0) + scale * (sum of
 * grad_out[i, :] over all i with tokens[i] == t), for every row t.  Sums are
 * held in fp32 in the order of i, in groups whose bounds depend on the tokens
 * alone: equal calls give equal bits.  Tokens outside [0, vocab) and those equal
 * to padding_idx (negative: none) contribute nothing.
 * workspace: la_embedding_grad_workspace(n, vocab, hidden) bytes, 16-byte aligned.
 */
uint64_t la_embedding_grad_workspace(uint64_t n, uint64_t vocab, uint64_t hidden);
int la_embedding_grad(int token_dtype, const void* tokens, uint64_t n, int g_dtype, const void* grad_out,
                      uint64_t grad_stride, int out_dtype, void* grad_weight, uint64_t vocab, uint64_t hidden,
                      uint64_t weight_stride, float scale, int64_t padding_idx, int accumulate, void* workspace,
                      uint64_t workspace_bytes, la_stream_t stream);

/*
 * z = x + residual (residual may be null: z = x), rstd = 1 / sqrt(mean(z^2) + eps),
 * y = z * rstd * weight, per row.  All in fp32 from the unrounded z; `summed`
 * (nullable) receives z and `out` y, each rounded once to dtype, `rstd` (nullable)
 * fp32.  With out_dtype LA_I8 or LA_F8E4M3, out holds y / scales[i] rounded to
 * nearest even, scales[i] = max|y| / 127 or / 448 (a row of zeros: scale 0 and zeros;
 * a row with an infinity or NaN: scale NaN and zeros).
 */
int la_rms_norm(int dtype, const void* x, uint64_t x_stride, const void* residual, uint64_t residual_stride,
                const void* weight, uint64_t n, uint64_t hidden, float eps, void* summed, uint64_t summed_stride,
                int out_dtype, void* out, uint64_t out_stride, float* scales, float* rstd, la_stream_t stream);

/*
 * From the gradient of y, grad_out, and of z, grad_summed (nullable): the gradient
 * of z (which is that of x and of residual) and of weight,
 *   grad_x = rstd * (g - u * mean(g * u)) + grad_summed,  u = z * rstd, g = grad_out * weight,
 *   grad_weight = (accumulate ? grad_weight : 0) + sum over rows of grad_out * u.
 * grad_weight (nullable) has type w_dtype.  Row partials are added in a fixed order.
 * workspace: la_rms_norm_grad_workspace(n, hidden) bytes, 16-byte aligned.
 */
uint64_t la_rms_norm_grad_workspace(uint64_t n, uint64_t hidden);
int la_rms_norm_grad(int dtype, const void* grad_out, uint64_t grad_out_stride, const void* summed,
                     uint64_t summed_stride, const float* rstd, const void* weight, const void* grad_summed,
                     uint64_t grad_summed_stride, uint64_t n, uint64_t hidden, void* grad_x, uint64_t grad_x_stride,
                     int w_dtype, void* grad_weight, int accumulate, void* workspace, uint64_t workspace_bytes,
                     la_stream_t stream);

/*
 * Softmax cross entropy of x [n, hidden] against weight [vocab, hidden]:
 * row_loss[i] = log(sum_v exp(s_iv)) - s_i,target, s = x weight^T, for every row
 * whose target is not ignore_index; ignored rows have loss 0, gradient 0, and are
 * never read.  loss = sum of the row losses, over the number of rows that are not
 * ignored with mean != 0 (0 where there are none).  A target outside [0, vocab)
 * makes its row's loss and gradient NaN.
 * With grads != 0 also grad_x = d loss / d x and grad_weight = (accumulate ?
 * grad_weight : 0) + d loss / d weight, both times *grad_scale (nullable: 1).
 * dtype (of x, weight, grad_x): LA_BF16 or LA_F16; grad_weight: that type or LA_F32.
 * Without gradients a tile of scores is held at a time.  With gradients the
 * softmax of piece_rows rows is held in 16 bits at a time (rounded up to a multiple of
 * 256; 0: of all; of 32768 at most), and up to half as much again or 64 MiB of partial sums of
 * grad_x.  Where the rows take more than one piece, grad_weight is summed in
 * fp32: where it lies if it is of fp32, else in the workspace; where that would take more
 * memory than the softmax of all rows, all rows are one piece.
 * workspace: la_linear_loss_workspace(call) bytes, 256-byte aligned.
 */
typedef struct {
    int dtype;
    const void* x;
    uint64_t n, hidden, x_stride;
    const void* weight;
    uint64_t vocab, weight_stride;
    const int64_t* targets;
    int64_t ignore_index;
    int mean;
    float* loss;              /* one fp32, nullable */
    float* row_loss;          /* n fp32, nullable */
    int grads;
    const float* grad_scale;  /* one fp32, nullable */
    void* grad_x;
    uint64_t grad_x_stride;
    int grad_weight_dtype;
    void* grad_weight;
    uint64_t grad_weight_stride;
    int accumulate;
    uint64_t piece_rows;
} la_linear_loss_t;

uint64_t la_linear_loss_workspace(const la_linear_loss_t* call);
int la_linear_loss(const la_linear_loss_t* call, void* workspace, uint64_t workspace_bytes, la_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SLIDEFORMER_AMD_MODEL_OPS_H */
