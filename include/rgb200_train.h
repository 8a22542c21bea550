/*
 * rgb200 - C ABI of the operators around the reproducible products of a training step  (librgb200.so)
 *
 * Same conventions as rgb200.h: plain device pointers and sizes, all work enqueued on the stream that is passed in (a
 * cudaStream_t cast to void*), nothing allocated, nothing kept between calls, cudaError_t codes as int
 * (0 = success, 1 = cudaErrorInvalidValue, 801 = cudaErrorNotSupported).  Calls that contain products report an expired bounded
 * wait through their workspace: rgb200_workspace_status reads it.  Sums of floats are taken in an order that depends
 * on the sizes alone, so the output bits depend on the inputs and the sizes, not on the stream, the call or the GPU.
 * Infinities and NaN stay visible: a row of an operand (of op(A), or a column of op(B)) that holds one makes every output of its product that it
 * takes part in NaN (the plain products of rgb200.h leave such outputs undefined), so a loss or a gradient that meets one is not finite;
 * rows of the cross entropy that do not count take no part in anything, whatever they hold.
 */
#ifndef RGB200_TRAIN_H
#define RGB200_TRAIN_H

#include <stddef.h>
#include <stdint.h>

#include "rgb200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------------------
 * Product with bias, activation and residual in its epilogue:
 *   Z = op(A) op(B) + bias,   C = act(Z) + residual
 * op(A) op(B) is the product of rgb200_gemm_fp32_ws bit for bit; each step behind it is one FP32 operation per value.
 * The reference's Linear adds its bias in a separate pass (repro_torch/repro_torch/layers.py:70-93).
 * bias [N], residual [M, N] (may be C itself) and pre_activation [M, N] (receives Z) may be NULL.  Activations: gelu is
 * z/2 (1 + erf(z / sqrt 2)), gelu_tanh z/2 (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))), silu z / (1 + exp(-z)).
 * Plan and workspace are those of rgb200_make_plan.  1: as rgb200_gemm_fp32_ws, or an unknown activation; 801: RGB200_ALGO_REFERENCE.
 * Slopes are those of the computed Z: relu's is 0 for Z <= 0, so a Z within the product's rounding of zero may pass or stop a gradient that
 * another product, rounded otherwise, would not.
 * rgb200_activation_backward: dZ = dY act'(Z) (dZ may be NULL, or dY itself) and db = column sums of dZ (may be NULL; the
 * workspace, of rgb200_activation_backward_workspace bytes, is needed for db alone).  Z may be NULL without an activation.  M and N are at most
 * 2^31 - 4097. */
enum { RGB200_ACT_NONE = 0, RGB200_ACT_RELU = 1, RGB200_ACT_SILU = 2, RGB200_ACT_GELU = 3, RGB200_ACT_GELU_TANH = 4 };
typedef struct rgb200_epilogue {
    const float* bias;
    const float* residual;
    float* pre_activation;
    int activation;
} rgb200_epilogue;
int rgb200_gemm_epilogue_fp32_ws(const float* A, const float* B, float* C, int M, int N, int K, const rgb200_config* cfg,
                                 const rgb200_epilogue* epilogue, void* workspace, size_t workspace_bytes, void* stream);
size_t rgb200_activation_backward_workspace(int M, int N);
int rgb200_activation_backward(const float* dY, const float* Z, float* dZ, float* db, int M, int N, int activation, void* workspace,
                               size_t workspace_bytes, void* stream);
/* The whole backward pass of Y = act(X W^T + bias) (+ residual, whose gradient is dY): with dZ = dY act'(Z), dX [M, K] = dZ W,
 * dW [N, K] = dZ^T X and db [N] = column sums of dZ; each of the three may be NULL.  The products are those of rgb200_gemm_fp32_ws
 * on dZ, bit for bit; dZ's digits for both come from one pass over it.  More than 1 056 751 rows at S = 3, which such a product does not take: dW
 * is the FP32 sum, in order, of the products of ranges of 2^20 rows.  Workspace: 256-byte aligned; 0 bytes: sizes not supported. */
size_t rgb200_linear_backward_workspace(int M, int N, int K, int activation, int slices);
int rgb200_linear_backward(const float* dY, const float* Z, const float* X, const float* W, float* dX, float* dW, float* db, int M, int N, int K,
                           int activation, int slices, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Cross entropy of the logits X W^T against targets, in pieces of the vocabulary: the [N, V] logits are never stored.
 * (The reference's cross entropy, repro_math_cuda/repro_softmax.cuh:8-49, takes stored logits.)
 * X [N, D], W [V, D], target [N] (int64).  Per row: lse = log sum exp(logits), target_rest = the probability of all words but the target
 * (summed over them, so that it keeps its digits in a confident row), nll = lse - logit of the target; 0 where the target is
 * ignore_index; NaN, and no gradient, where it is any other value outside 0 .. V - 1.  Reductions: NONE leaves nll, SUM and
 * MEAN write *loss (MEAN divides by the number of rows that are not ignored, at least 1).
 * SUM and MEAN also write *inv_count, what the rows' weights are multiplied by (MEAN: the reciprocal count; SUM: 1).
 * Backward: dloss points to one value (SUM, MEAN) or N of them (NONE); lse, target_rest and inv_count are the forward call's.
 *   dX = sum_j g p_j W_j - g W_target,  dW = sum_i g_i (p_i - onehot_i) x_i,  g the row's weight; either may be NULL.
 * The logits are the library's products (S = `slices`); sums are taken in an order that depends on the sizes and targets
 * alone (dW's, beyond 1 056 751 rows at S = 3, over ranges of 2^20 rows).  D at most 105472 (S = 3).  Workspaces: 256-byte aligned, rgb200_linear_xent_workspace bytes (0: sizes not supported). */
enum { RGB200_REDUCE_NONE = 0, RGB200_REDUCE_MEAN = 1, RGB200_REDUCE_SUM = 2 };
size_t rgb200_linear_xent_workspace(int N, int V, int D, int slices, int backward);
int rgb200_linear_xent_forward(const float* X, const float* W, const long long* target, long long ignore_index, int reduction, int N, int V,
                               int D, int slices, float* loss, float* nll, float* lse, float* target_rest, float* inv_count,
                               void* workspace, size_t workspace_bytes, void* stream);
int rgb200_linear_xent_backward(const float* X, const float* W, const long long* target, long long ignore_index, int reduction, int N, int V,
                                int D, int slices, const float* lse, const float* target_rest, const float* inv_count, const float* dloss,
                                float* dX, float* dW, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------
 * AdamW over many tensors in one launch, moments in FP32 or as 8-bit codes.
 * Stands beside the reference's Adam / AdamW (repro_nn_cuda/repro_nn.cuh:12-21), which takes one FP32 tensor per call.
 * Per value, every operation an IEEE single operation in this order (constants in parentheses formed in
 * double, rounded once), n the step's number counted from 1:
 *   p1 = p (1 - lr wd);  m' = m b1 + g (1 - b1);  v' = v b2 + (g g)(1 - b2)
 *   p' = p1 - (m' / (sqrt(v') (1 / sqrt(1 - b2^n)) + eps)) (lr / (1 - b1^n))
 * so the result does not depend on how tensors are cut, ordered or spread over calls, streams or GPUs.
 * 8-bit states: 256 consecutive values of a tensor share one FP32 scale (the largest magnitude of the block);
 * a first moment is an int8 code q standing for (q/127) |q/127| scale, a second moment a uint8 code standing for
 * (q/255)^4 scale, rounded to the nearest code in q, a non-zero second moment never to code 0.  A block that
 * holds a value that is not finite gets a NaN scale.
 * Asynchronous on `stream` and allocation-free.  The tensors of one call must not overlap.
 * 1 (invalid value): a null pointer with count > 0, a negative count, betas outside [0, 1), negative or NaN
 * lr / eps / weight decay, step < 1 without device_step, state_bits not 8 or 32. */
typedef struct rgb200_adamw_tensor {
    float* param;
    const float* grad;
    void* exp_avg;            /* float[count], or int8[count] codes */
    void* exp_avg_sq;         /* float[count], or uint8[count] codes */
    float* exp_avg_scale;     /* 8-bit states: float[ceil(count / 256)]; else ignored */
    float* exp_avg_sq_scale;
    long long count;
} rgb200_adamw_tensor;
typedef struct rgb200_adamw_hyper {
    double lr, beta1, beta2, eps, weight_decay;
    long long step;           /* this step's number, from 1; ignored with device_step */
    long long* device_step;   /* or NULL: device word with the number of steps done; read, then advanced by this call
                               * (for steps captured into a CUDA graph) */
    int state_bits;           /* 32 or 8 */
} rgb200_adamw_hyper;
int rgb200_adamw_step(const rgb200_adamw_tensor* tensors, int count, const rgb200_adamw_hyper* hyper, void* stream);
/* The values that 8-bit states stand for, written to param (first moments) and grad (second moments), and the
 * reverse: codes and scales of the values found there.  Used for checkpoints that either state width can load. */
int rgb200_adamw_states_read(const rgb200_adamw_tensor* tensors, int count, void* stream);
int rgb200_adamw_states_write(const rgb200_adamw_tensor* tensors, int count, void* stream);

/* ------------------------------------------------------------------------------------------------
 * The norm behind a block, its gate, the residual stream and the norm in front of the next block (no counterpart in
 * the reference).  All tensors FP32, rows of `dim` contiguous values:
 *   u = post_weight * N(y)  (u = y when post_weight is NULL)      r = scale x + gate * u      h = weight * N(r) + bias
 * and h = weight * N(x) + bias when y is NULL (r is then not written).  N subtracts the mean (layer kind) and divides by
 * sqrt(mean of squares + eps).  gate holds `groups` rows of `dim` values, each for rows / groups consecutive rows; with
 * groups 1 it is one value a channel.
 * stats (float[4 * rows]; forward: may be NULL) carries the rows' means and reciprocal deviations to the backward call, which
 * takes the gradients dr (of r from elsewhere; may be NULL) and dh, and writes those outputs that are not NULL: dx[rows, dim],
 * dy, dweight[dim], dbias[dim], dpost_weight[dim], dgate[groups, dim].  Without y, r is x: r is not read, and dr (of x from the
 * residual stream) is added to dx as it is.
 * Sums are taken in an order that depends on (rows, dim, groups) alone.  Asynchronous and allocation-free; dim at most 8192,
 * groups at most 2^30.
 * The workspace (16-byte aligned) may be reused by any later call on the same stream.
 * 1 (invalid value): sizes outside those limits, rows not a multiple of groups, negative or NaN eps, post_weight or gate or
 * dy without y, gradients of absent tensors, missing tensors, a short workspace. */
enum { RGB200_NORM_RMS = 0, RGB200_NORM_LAYER = 1 };
typedef struct rgb200_block_norm {
    int rows, dim, groups, kind;
    float scale, eps;
    const float *x, *y, *weight, *bias, *post_weight, *gate;
    float *r, *h, *stats;
    const float *dr, *dh;
    float *dx, *dy, *dweight, *dbias, *dpost_weight, *dgate;
} rgb200_block_norm;
int rgb200_block_norm_forward(const rgb200_block_norm* norm, void* stream);
size_t rgb200_block_norm_backward_workspace(int rows, int dim, int groups);
int rgb200_block_norm_backward(const rgb200_block_norm* norm, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RGB200_TRAIN_H */
