// Kernels around the products of the linear cross entropy (see rgb200_loss.cu for the sequence).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "rgb200_math.cuh"

namespace rgb200 {

constexpr int XENT_ROWS = 32, XENT_WARPS = 16;

// (maximum, sum of exp(value - maximum)) of two sets of values; an empty set is (-inf, 0), one of NaN alone (-inf, NaN).
__device__ __forceinline__ float2 lse_join(float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x);
    if (top == -INFINITY) return make_float2(top, a.y + b.y);
    return make_float2(top, a.y * expf(a.x - top) + b.y * expf(b.x - top));
}

// One vocabulary piece's partial statistics [parts][rows] joined into the rows' running ones: a CTA owns 32 rows (lanes), warp k joins
// parts k, k + 16, ... in order, then the warps' results in order.  last: also log-sum-exp and loss of each row, and in place of its target's logit
// the probability of all words but the target.
//
// The maximum m is over all words, the sum over all but the target.  A confident row's loss and its target's gradient are as small as
// the others' probability 1 - p; from p or from the log-sum-exp they would come out as a difference of numbers near 1 or near the logits: with logits
// near 60 and 1 - p = 1e-5 a fifth of the value would be rounding, near 300 all of it.  As a sum of the others nothing cancels.
static __global__ void __launch_bounds__(32 * XENT_WARPS)
xent_join_kernel(const float2* __restrict__ parts, int count, float2* running, int rows, bool first, bool last, const long long* __restrict__ target,
                 long long ignore, int vocab, float* target_rest, float* lse, float* nll) {
    __shared__ float2 joined[XENT_WARPS][XENT_ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * XENT_ROWS + lane;
    float2 s = make_float2(-INFINITY, 0.0f);
    if (row < rows) {
#pragma unroll 4
        for (int i = warp; i < count; i += XENT_WARPS) s = lse_join(s, parts[(size_t)i * rows + row]);
    }
    joined[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || row >= rows) return;
    for (int k = 1; k < XENT_WARPS; ++k) s = lse_join(s, joined[k][lane]);
    if (!first) s = lse_join(running[row], s);
    running[row] = s;
    if (!last) return;
    const long long t = target[row];
    const bool word = t >= 0 && t < vocab;
    const float z = word ? target_rest[row] : 0.0f, total = word ? s.y + expf(z - s.x) : s.y;
    lse[row] = s.x + logf(total);
    target_rest[row] = s.y / total;
    // a target outside the vocabulary makes the row's loss NaN; an ignored one leaves it 0.  Where the target is the largest, total is 1 + s.y;
    // elsewhere it is above 1, and all terms are positive
    nll[row] = t == ignore ? 0.0f : !word ? __int_as_float(0x7FC00000) : (s.x - z) + (z == s.x ? log1pf(s.y) : logf(total));
}

// Sum of the rows' losses (in double, thread t adding rows t, t + 1024, ..., then a tree) over the number of rows that count.
// inv_count receives 1 / max(1, rows that count) for the mean, 1 for the sum.
static __global__ void __launch_bounds__(1024)
xent_reduce_kernel(const float* __restrict__ nll, const long long* __restrict__ target, long long ignore, int rows, bool mean, float* loss, float* inv_count) {
    __shared__ double sums[1024];
    __shared__ int counts[1024];
    double s = 0.0;
    int n = 0;
    for (int i = threadIdx.x; i < rows; i += 1024) {
        s += (double)nll[i];
        n += target[i] != ignore;
    }
    sums[threadIdx.x] = s;
    counts[threadIdx.x] = n;
    __syncthreads();
    for (int w = 512; w > 0; w >>= 1) {
        if (threadIdx.x < w) {
            sums[threadIdx.x] += sums[threadIdx.x + w];
            counts[threadIdx.x] += counts[threadIdx.x + w];
        }
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    const double many = mean ? (double)(counts[0] > 1 ? counts[0] : 1) : 1.0;
    *loss = (float)(sums[0] / many);
    *inv_count = (float)(1.0 / many);
}

// One CTA a row: the row's weight g (the loss's gradient, over the number of rows for the mean; 0 for rows that do not count) and its
// target's coefficient (p - 1) g, from the sum of the others' probabilities; for the target word its first row and the complement of its last one (integer minima of words
// that start at 0x7F7F7F7F: any order); and dX's start, coefficient times the target's row of W, to which the pieces' products are added.
static __global__ void __launch_bounds__(128)
xent_rows_kernel(const long long* __restrict__ target, long long ignore, int vocab, int dim, const float* __restrict__ target_rest, const float* __restrict__ dloss, bool per_row, const float* __restrict__ inv_count,
                 const float* __restrict__ W, float* weight, float* coefficient, int* first, int* not_last, float* dX) {
    const int i = blockIdx.x;
    const long long t = target[i];
    const bool counts = t != ignore && t >= 0 && t < vocab;
    const float g = counts ? (per_row ? dloss[i] : dloss[0] * *inv_count) : 0.0f;
    const float c = counts ? -target_rest[i] * g : 0.0f;
    if (threadIdx.x == 0) {
        weight[i] = g;
        coefficient[i] = c;
        if (counts) {
            atomicMin(first + t, i);
            atomicMin(not_last + t, ~i);
        }
    }
    if (!dX) return;
    const float* w = W + (size_t)(counts ? t : 0) * dim;
#pragma unroll 4
    for (int k = threadIdx.x; k < dim; k += 128) dX[(size_t)i * dim + k] = c != 0.0f ? c * w[k] : 0.0f;
}

// dW[t] += sum over the rows with target t of coefficient * x, in two kernels.  The first gives a warp to each row: it adds the row itself
// where no other has its target, and lists it where it is the first of several (in any order: the listed words are independent).
static __global__ void __launch_bounds__(256)
xent_single_dw_kernel(const long long* __restrict__ target, const float* __restrict__ coefficient, const float* __restrict__ X, const int* __restrict__ first,
                      const int* __restrict__ not_last, int rows, int vocab, int dim, float* dW, int* list, int* listed) {
    const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const long long t = target[row];
    if (t < 0 || t >= vocab || first[t] != row) return;                     // ignored rows were never entered in first
    if (~not_last[t] != row) {
        if (lane == 0) list[atomicAdd(listed, 1)] = row;
        return;
    }
    const float c = coefficient[row];
    const float* x = X + (size_t)row * dim;
    float* w = dW + (size_t)t * dim;
#pragma unroll 4
    for (int k = lane; k < dim; k += 32) w[k] += c * x[k];
}

// The second takes the listed words, 128 columns at a time.  Its eight warps take the range from the word's first to its last row in eight
// equal stretches, each adding its rows in order, then the warps' sums are added in order: the order depends on the targets alone.
constexpr int XENT_DW_COLS = 128;
static __global__ void __launch_bounds__(256)
xent_repeated_dw_kernel(const long long* __restrict__ target, const float* __restrict__ coefficient, const float* __restrict__ X,
                        const int* __restrict__ not_last, int dim, float* dW, const int* __restrict__ list, const int* __restrict__ listed) {
    __shared__ float sums[8][XENT_DW_COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, strips = (dim + XENT_DW_COLS - 1) / XENT_DW_COLS;
    const long long items = (long long)*listed * strips;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int row = list[item / strips], strip = (int)(item % strips);
        const long long t = target[row];
        const int last = ~not_last[t];
        const int stretch = (last - row) / 8 + 1, begin = row + warp * stretch;
        const int end = begin + stretch < last + 1 ? begin + stretch : last + 1;
        const int col0 = strip * XENT_DW_COLS + lane;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int base = begin; base < end; base += 32) {
            const int i = base + lane;
            unsigned hits = __ballot_sync(0xFFFFFFFFu, i < end && target[i] == t);
            while (hits) {                                   // four rows' loads in flight, added in order
                float c[4], x[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool some = hits != 0;
                    const int k = some ? base + __ffs(hits) - 1 : row;
                    hits &= hits - 1;
                    c[i] = some ? coefficient[k] : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = some && col0 + 32 * j < dim ? X[(size_t)k * dim + col0 + 32 * j] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[j] += c[i] * x[i][j];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[warp][lane + 32 * j] = s[j];
        __syncthreads();
        const int c = threadIdx.x, col = strip * XENT_DW_COLS + c;
        if (c < XENT_DW_COLS && col < dim) {
            float total = sums[0][c];
#pragma unroll
            for (int k = 1; k < 8; ++k) total += sums[k][c];
            dW[(size_t)t * dim + col] += total;
        }
        __syncthreads();
    }
}

}  // namespace rgb200
