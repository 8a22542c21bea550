// Epilogues of the tcgen05 GEMM kernel (rgb200_mma.cuh) and of the rounding kernel behind K ranges:
//
//   EPI_LINEAR   y = act(c + bias[col]) + residual[row][col], with c + bias stored beside it on request.
//   EPI_LSE      per row: m = max over the tile's columns, s = sum exp(c - m) over all but the row's target word; of c only the target's is stored.
//   EPI_PROB     row_scale[row] * exp(c - lse[row]), zero at the row's target word.
//
// c is the product rounded once to FP32, as the plain entry points return it; every step after it is one FP32 operation in a
// fixed order, so the bits do not depend on the tiling (EPI_LSE: on the tile width alone).  c is NaN where its row or column is marked
// as not finite, and the maxima left for a split keep NaN.
//
// Why here: an output costs 4 bytes of HBM written by the product and 8 more for every elementwise pass behind it.  In
// the kernel the extra work of a thread (16 or 32 columns of one row) overlaps the next tile's MMAs, which take about 1150 clocks for each
// 128 values of k; the residual and the bias are requested before the wait for the accumulators.
#pragma once
#include "rgb200_mma.cuh"
#include "rgb200_prepass.cuh"

namespace rgb200 {

constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_COUNT = 5;

// 2 sqrt(2 / pi), and that times 0.044715; gelu_tanh(z) = z / (1 + exp(-(G1 z + G3 z^3))), which is 0.5 z (1 + tanh(half of it)) without
// the cancellation of 1 + tanh on the negative side.
constexpr float GELU_G1 = 1.5957691216057308f, GELU_G3 = 0.0713548162726009f;
// The same for a power of two, log2(e) folded into the constants: exp(-t) = 2^(-t log2 e), one multiplication and rounding less.
constexpr float GELU_L1 = 2.302208198f, GELU_L3 = 0.102943240f;
__device__ __forceinline__ float exp2_fast(float x) {           // within 2 ulp
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float SQRT_HALF = 0.7071067811865476f, INV_SQRT_2PI = 0.3989422804014327f;

template <int ACT>
__device__ __forceinline__ float activation(float z) {
    if (ACT == ACT_RELU) return z <= 0.0f ? 0.0f : z;
    if (ACT == ACT_SILU) return z / (1.0f + expf(-z));
    if (ACT == ACT_GELU) return 0.5f * z * (1.0f + erff(z * SQRT_HALF));
    if (ACT == ACT_GELU_TANH) return z / (1.0f + exp2_fast(-z * (GELU_L1 + GELU_L3 * (z * z))));
    return z;
}

// Derivative of the activation.  Where exp overflows the sigmoid is 0 and the products with it are 0 for any finite z: gelu_tanh's inner
// slope, a cube's, would overflow beyond 1e13 and is taken at 64 there, where p (1 - p) is 0 already.
template <int ACT>
__device__ __forceinline__ float activation_slope(float z) {
    if (ACT == ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
    if (ACT == ACT_SILU) {
        const float p = 1.0f / (1.0f + expf(-z));
        return p * (1.0f + z * (1.0f - p));
    }
    if (ACT == ACT_GELU) return 0.5f * (1.0f + erff(z * SQRT_HALF)) + z * (expf(-0.5f * (z * z)) * INV_SQRT_2PI);
    if (ACT == ACT_GELU_TANH) {
        const float q = z * z, p = 1.0f / (1.0f + exp2_fast(-z * (GELU_L1 + GELU_L3 * q)));
        const float c = fminf(fmaxf(z, -64.0f), 64.0f);
        return p + (p * (1.0f - p)) * (c * (GELU_G1 + 3.0f * GELU_G3 * (c * c)));
    }
    return 1.0f;
}

// Runs f with the activation as a compile-time constant: one uniform branch instead of one per value.
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
    switch (act) {
        case ACT_RELU: f(std::integral_constant<int, ACT_RELU>()); break;
        case ACT_SILU: f(std::integral_constant<int, ACT_SILU>()); break;
        case ACT_GELU: f(std::integral_constant<int, ACT_GELU>()); break;
        case ACT_GELU_TANH: f(std::integral_constant<int, ACT_GELU_TANH>()); break;
        default: f(std::integral_constant<int, ACT_NONE>()); break;
    }
}

__device__ __forceinline__ void ld_global_256(const float* p, float (&v)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void st_global_256(float* p, const float (&v)[8]) {
    st_global_256(reinterpret_cast<uint32_t*>(p), __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]),
                  __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}

template <int CPT>
struct EpilogueRow<EPI_LINEAR, CPT> {
    float res[CPT];
    bool sectors;               // the thread's columns are whole 32-byte sectors of C, residual and pre

    __device__ __forceinline__ void request(const GemmParams& P, int row, bool row_ok, int col0, float* slot, int lane) {
        for (int c = lane; c < CPT; c += 32) slot[c] = P.epi.bias && col0 + c < P.N ? __ldg(P.epi.bias + col0 + c) : 0.0f;
        const size_t at = (size_t)row * P.N + col0;
        const uintptr_t bits = reinterpret_cast<uintptr_t>(P.C + at) | (P.epi.residual ? reinterpret_cast<uintptr_t>(P.epi.residual + at) : 0) |
                               (P.epi.pre ? reinterpret_cast<uintptr_t>(P.epi.pre + at) : 0);
        sectors = (bits & 31) == 0 && col0 + CPT <= P.N;
        if (!row_ok || !P.epi.residual) return;
        if (sectors) {
#pragma unroll
            for (int j = 0; j < CPT; j += 8) {
                float v[8];
                ld_global_256(P.epi.residual + at + j, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) res[j + i] = v[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < CPT; ++j) res[j] = col0 + j < P.N ? P.epi.residual[at + j] : 0.0f;
        }
    }

    template <class Values>
    __device__ __forceinline__ void finish(const GemmParams& P, int row, bool row_ok, int col0, int, const float* slot, Values values) {
        if (!row_ok) return;
        const size_t at = (size_t)row * P.N + col0;
        with_activation(P.epi.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < CPT; j += 8) {
                float z[8], y[8];
                values(j, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (P.epi.bias) z[i] += slot[j + i];
                    y[i] = activation<decltype(act)::value>(z[i]);
                    if (P.epi.residual) y[i] += res[j + i];
                }
                if (sectors) {
                    if (P.epi.pre) st_global_256(P.epi.pre + at + j, z);
                    st_global_256(P.C + at + j, y);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (col0 + j + i >= P.N) break;
                        if (P.epi.pre) P.epi.pre[at + j + i] = z[i];
                        P.C[at + j + i] = y[i];
                    }
                }
            }
        });
    }
};

// Column of the row's target among the thread's columns, or a value outside 0 .. CPT - 1.
__device__ __forceinline__ int target_column(const GemmParams& P, int row, int col0) {
    const long long t = P.epi.target[row] - P.epi.first_word - col0;
    return t < 0 || t > 0x7FFFFFFF ? -1 : (int)t;
}

template <int CPT>
struct EpilogueRow<EPI_LSE, CPT> {
    int target;

    __device__ __forceinline__ void request(const GemmParams& P, int row, bool row_ok, int col0, float*, int) {
        target = row_ok ? target_column(P, row, col0) : -1;
    }

    template <class Values>
    __device__ __forceinline__ void finish(const GemmParams& P, int row, bool row_ok, int col0, int part, const float*, Values values) {
        if (!row_ok) return;
        float v[CPT], top = -INFINITY, sum = 0.0f, hit = 0.0f;
#pragma unroll
        for (int j = 0; j < CPT; j += 8) {
            float c[8];
            values(j, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[j + i] = col0 + j + i < P.N ? c[i] : -INFINITY;          // the first column is always inside, so top is finite
                top = fmaxf(top, v[j + i]);
                if (j + i == target) {                                     // kept apart from the sum: see xent_join_kernel
                    hit = c[i];
                    v[j + i] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < CPT; ++j) sum += expf(v[j] - top);
        P.epi.lse_parts[(size_t)part * P.M + row] = make_float2(top, sum);
        if (target >= 0 && target < CPT && col0 + target < P.N) P.epi.target_logit[row] = hit;
    }
};

template <int CPT>
struct EpilogueRow<EPI_PROB, CPT> {
    int target;
    float lse, scale;

    __device__ __forceinline__ void request(const GemmParams& P, int row, bool row_ok, int col0, float*, int) {
        target = row_ok ? target_column(P, row, col0) : -1;
        lse = row_ok ? __ldg(P.epi.lse + row) : 0.0f;
        scale = row_ok ? __ldg(P.epi.row_scale + row) : 0.0f;
    }

    template <class Values>
    __device__ __forceinline__ void finish(const GemmParams& P, int row, bool row_ok, int col0, int, const float*, Values values) {
        float* dst = P.C + (size_t)row * P.epi.ldc + col0;
        const bool sectors = row_ok && (reinterpret_cast<uintptr_t>(dst) & 31) == 0 && col0 + CPT <= P.epi.ldc;      // zeros behind the last word
        float row_top = 0.0f;
        unsigned col_top = 0;
        static_assert(CPT <= 32, "one column a lane");
#pragma unroll
        for (int j = 0; j < CPT; j += 8) {
            float p[8];
            values(j, p);
#pragma unroll
            for (int i = 0; i < 8; ++i) {          // a row without a weight takes no part, whatever its logits are
                p[i] = j + i == target || scale == 0.0f || col0 + j + i >= P.N ? 0.0f : __expf(p[i] - lse) * scale;
                row_top = max_nan(row_top, fabsf(p[i]));
            }
            if (P.epi.col_max) {                   // rows that do not exist have no weight and join as zeros
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fabsf(p[i])));     // NaN is the largest
                    if ((threadIdx.x & 31) == j + i) col_top = top;
                }
            }
            if (sectors) st_global_256(dst + j, p);
            else if (row_ok) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (col0 + j + i < P.N) dst[j + i] = p[i];
            }
        }
        if (P.epi.row_max && row_ok) atomicMax(P.epi.row_max + row, __float_as_uint(row_top));
        if (P.epi.col_max) {
            const int c = threadIdx.x & 31;
            if (c < CPT && col0 + c < P.N) atomicMax(P.epi.col_max + col0 + c, col_top);
        }
    }
};

// The same on values that a K-range product left as INT64 sums: see round_partial_kernel.  Four neighbours per thread when
// VEC, which the host sets from N and the addresses.
template <bool VEC>
static __global__ void __launch_bounds__(256)
round_partial_linear_kernel(const long long* __restrict__ partial, int parts, const int* __restrict__ ea, const int* __restrict__ eb, int M, int N,
                            float* C, int e0, const EpilogueParams E) {
    constexpr int W = VEC ? 4 : 1;
    const size_t total = (size_t)M * N;
    with_activation(E.act, [&](auto act) {
        for (size_t idx = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * W; idx < total; idx += (size_t)gridDim.x * blockDim.x * W) {
            long long t[W];
#pragma unroll
            for (int j = 0; j < W; ++j) t[j] = 0;
            for (int p = 0; p < parts; ++p) {
#pragma unroll
                for (int j = 0; j < W; ++j) t[j] += partial[(size_t)p * total + idx + j];
            }
            const int r = (int)(idx / N), c = (int)(idx - (size_t)r * N);
            const int e_r = ea[r] + e0;
            float z[W], y[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                z[j] = bits_f32(round_or_nan(t[j], e_r + eb[c + j]));
                if (E.bias) z[j] += E.bias[c + j];
                y[j] = activation<decltype(act)::value>(z[j]);
            }
            if (VEC) {
                if (E.residual) {
                    const float4 q = *reinterpret_cast<const float4*>(E.residual + idx);
                    y[0] += q.x; y[W > 1 ? 1 : 0] += q.y; y[W > 2 ? 2 : 0] += q.z; y[W > 3 ? 3 : 0] += q.w;
                }
                if (E.pre) *reinterpret_cast<float4*>(E.pre + idx) = make_float4(z[0], z[W > 1 ? 1 : 0], z[W > 2 ? 2 : 0], z[W > 3 ? 3 : 0]);
                *reinterpret_cast<float4*>(C + idx) = make_float4(y[0], y[W > 1 ? 1 : 0], y[W > 2 ? 2 : 0], y[W > 3 ? 3 : 0]);
            } else {
                if (E.residual) y[0] += E.residual[idx];
                if (E.pre) E.pre[idx] = z[0];
                C[idx] = y[0];
            }
        }
    });
}

// ------------------------------------------------------------------------------------------
// Backward of the epilogue: dZ = dY * act'(Z) and the bias gradient db = column sums of dZ, one pass (HBM: 12 bytes a value, 4 when
// there is no activation and only db is formed).  A CTA owns 128 columns of a range of rows; each of its eight warps adds
// every eighth row of the range in order, then the warps' sums and last the ranges' are added in order: an order that depends on
// (M, N) alone.  Lane columns: neighbours in quads when N % 4 == 0 (an unaligned base only changes how they are loaded).
// ------------------------------------------------------------------------------------------
constexpr int ACTB_COLS = 128, ACTB_WARPS = 8;

struct ActBackwardParams {
    const float *dy, *z;
    float *dz;                  // null: only the column sums
    float *parts;               // [ranges][N], or null without a bias gradient
    unsigned *row_max, *col_max;        // [M], [N]: the bits of dZ's largest magnitudes are joined in (zeroed by the caller), or null
    int M, N, act, rows_per_range, wide;
};

template <int V>
static __global__ void __launch_bounds__(32 * ACTB_WARPS)
activation_backward_kernel(const ActBackwardParams P) {
    __shared__ float sums[ACTB_WARPS][ACTB_COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = blockIdx.y * P.rows_per_range;
    const int end = P.M - first < P.rows_per_range ? P.M : first + P.rows_per_range;
    int col[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) col[j] = blockIdx.x * ACTB_COLS + (V == 4 ? lane * 4 + j : j * 32 + lane);
    const bool wide = V == 4 && P.wide;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, top[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    with_activation(P.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        constexpr int BATCH = 4;            // rows whose loads are in flight together (dZ may be dY, so none moves over a store)
        for (int row0 = first + warp; row0 < end; row0 += BATCH * ACTB_WARPS) {
            float d[BATCH][4], z[BATCH][4];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int row = row0 + i * ACTB_WARPS;
                const size_t at = (size_t)row * P.N;
#pragma unroll
                for (int j = 0; j < 4; ++j) d[i][j] = z[i][j] = 0.0f;
                if (row >= end) continue;
                if (wide) {
                    if (col[0] < P.N) {
                        const float4 q = *reinterpret_cast<const float4*>(P.dy + at + col[0]);
                        d[i][0] = q.x; d[i][1] = q.y; d[i][2] = q.z; d[i][3] = q.w;
                        if (ACT != ACT_NONE) {
                            const float4 t = *reinterpret_cast<const float4*>(P.z + at + col[0]);
                            z[i][0] = t.x; z[i][1] = t.y; z[i][2] = t.z; z[i][3] = t.w;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col[j] < P.N) {
                            d[i][j] = P.dy[at + col[j]];
                            if (ACT != ACT_NONE) z[i][j] = P.z[at + col[j]];
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int row = row0 + i * ACTB_WARPS;
                if (row >= end) break;                              // uniform over the warp
                const size_t at = (size_t)row * P.N;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (ACT != ACT_NONE) d[i][j] = d[i][j] * activation_slope<ACT>(z[i][j]);
                    s[j] += d[i][j];
                    top[j] = max_nan(top[j], fabsf(d[i][j]));
                }
                if (P.dz) {
                    if (wide) {
                        if (col[0] < P.N) *reinterpret_cast<float4*>(P.dz + at + col[0]) = make_float4(d[i][0], d[i][1], d[i][2], d[i][3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (col[j] < P.N) P.dz[at + col[j]] = d[i][j];
                    }
                }
                if (P.row_max) {
                    const float m = max_nan(max_nan(fabsf(d[i][0]), fabsf(d[i][1])), max_nan(fabsf(d[i][2]), fabsf(d[i][3])));
                    const unsigned all = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m));
                    if (lane == 0) atomicMax(P.row_max + row, all);
                }
            }
        }
    });
    if (P.col_max) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[warp][col[j] - blockIdx.x * ACTB_COLS] = top[j];
        __syncthreads();
        const int c = threadIdx.x, out = blockIdx.x * ACTB_COLS + c;
        if (c < ACTB_COLS && out < P.N) {
            float m = sums[0][c];
#pragma unroll
            for (int k = 1; k < ACTB_WARPS; ++k) m = max_nan(m, sums[k][c]);
            atomicMax(P.col_max + out, __float_as_uint(m));
        }
        __syncthreads();
    }
    if (!P.parts) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[warp][col[j] - blockIdx.x * ACTB_COLS] = s[j];
    __syncthreads();
    const int c = threadIdx.x, out = blockIdx.x * ACTB_COLS + c;
    if (c < ACTB_COLS && out < P.N) {
        float t = sums[0][c];
#pragma unroll
        for (int k = 1; k < ACTB_WARPS; ++k) t += sums[k][c];
        P.parts[(size_t)blockIdx.y * P.N + out] = t;
    }
}

// Column sums of the ranges' sums, [ranges][N] -> [N]: a CTA owns 32 columns, warp k adds ranges k, k + 8, ... in order, then the warps' sums.
static __global__ void __launch_bounds__(256)
range_sums_kernel(const float* __restrict__ parts, int ranges, int N, float* __restrict__ out) {
    __shared__ float sums[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < N) {
#pragma unroll 4
        for (int i = warp; i < ranges; i += 8) s += parts[(size_t)i * N + col];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || col >= N) return;
    for (int k = 1; k < 8; ++k) s += sums[k][lane];
    out[col] = s;
}

}  // namespace rgb200
