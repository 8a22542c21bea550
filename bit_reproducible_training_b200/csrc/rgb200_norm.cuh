// The norm behind a block, its gate, the residual stream and the norm in front of the next block, in one pass over the
// rows, and the gradients of all of it in another.
//
//   u = w' * N(y)                      (post norm; u = y without one)
//   r = s x + g * u                    (g: none, one value a channel, or one a channel for each group of rows)
//   h = w * N(r) + b                   (r = x when there is no y)
// N(t) = (t - mean) * rstd with rstd = 1 / sqrt(mean((t - mean)^2) + eps); the RMS kind leaves the mean out.
//
// Backward, with R = gradient of r from the residual stream, H = gradient of h, t^ the normed rows and
// N'(t^, rstd, q) = rstd (q - t^ mean(q t^) - mean(q)) (the RMS kind without the last term):
//   D  = R + N'(r^, rstd, w H)         dx = s D  (D when there is no y)
//   dy = N'(y^, rstd', w' g D)         (or g D without a post norm)
//   dw = sum_rows H r^,  db = sum_rows H,  and with Q = sum_rows D y^ (D y without a post norm) over the rows of a group,
//   dw' = sum_groups g Q,  dg = w' Q.
//
// Bound: HBM (measured, 8192 x 4096 with post norm and gate: forward 84 us = 6.4 TB/s).  A row is read once and stays in registers: its sums are taken from there (for the layer kind the mean first,
// then the squared differences, so that a large mean costs no precision).
//
// Order of the sums, which fixes the bits: a thread adds its values of a row in column order, a warp joins lanes by a
// butterfly, the warps' sums are added in order.  Lanes and columns are assigned by the row length alone.  Column sums
// (backward) add the rows of a fixed range in order (NormParams::rows_per_part, chosen from the sizes alone), then the ranges in order.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "rgb200_math.cuh"

namespace rgb200 {

constexpr int NORM_VALUES = 8;                   // values of a row per thread
constexpr int NORM_MAX_DIM = 1024 * NORM_VALUES;
constexpr int NORM_MAX_GROUPS = 1 << 30;         // the sums over the groups count in strides of 32 bits

struct NormParams {
    const float *x, *y, *w, *b, *pw, *gate;      // y, b, pw, gate may be null (pw, gate only with y)
    float *r, *h;                                // r null when y is
    float* stats;                                // [4][rows]: mean, rstd of r, mean, rstd of y (null: not kept)
    int rows, dim, group_rows;                   // group_rows: rows that share a row of the gate
    int layer;                                   // 1: layer norm, 0: RMS norm
    int wide;                                    // every row starts at a 16-byte boundary
    float scale, eps;
    // backward
    const float *dr, *dh;                        // dr may be null
    float *dx, *dy;
    float* parts;                                // [parts][3][dim] column sums of row ranges: H r^, H, D y^ (or D y)
    int rows_per_part, parts_per_group, parts_total, groups;
    float *dw, *db, *dpw, *dgate;                // null: not wanted
};

// Column of value j of a thread: quads of neighbours where the row length allows it, so that a thread moves 16 bytes at
// once; the assignment goes by the length alone (an unaligned base only changes how the same columns are loaded).
template <int TPR, int V>
__device__ __forceinline__ int norm_column(int lane, int j) { return V == 4 ? ((j >> 2) * TPR + lane) * 4 + (j & 3) : j * TPR + lane; }

template <int TPR, int V>
__device__ __forceinline__ void norm_load(const float* row, int dim, int lane, bool wide, float (&v)[NORM_VALUES]) {
    if (V == 4 && wide) {
#pragma unroll
        for (int c = 0; c < NORM_VALUES / 4; ++c) {
            const int col = (c * TPR + lane) * 4;
            const float4 q = col < dim ? *reinterpret_cast<const float4*>(row + col) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * c] = q.x; v[4 * c + 1] = q.y; v[4 * c + 2] = q.z; v[4 * c + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) {
            const int col = norm_column<TPR, V>(lane, j);
            v[j] = col < dim ? row[col] : 0.0f;
        }
    }
}
template <int TPR, int V>
__device__ __forceinline__ void norm_store(float* row, int dim, int lane, bool wide, const float (&v)[NORM_VALUES]) {
    if (V == 4 && wide) {
#pragma unroll
        for (int c = 0; c < NORM_VALUES / 4; ++c) {
            const int col = (c * TPR + lane) * 4;
            if (col < dim) *reinterpret_cast<float4*>(row + col) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) {
            const int col = norm_column<TPR, V>(lane, j);
            if (col < dim) row[col] = v[j];
        }
    }
}

// Sums over the TPR threads of a row, the same value in every thread.  A CTA may hold several rows, each with its own named
// barrier and its own slots; consecutive calls use the two sets of slots in turn, so that one barrier a call is enough: a
// warp writes a set again only after every warp has passed the barrier of the call in between.
constexpr int NORM_SLOTS = 2 * 2 * 32;           // floats per row of a CTA: two sets, two sums, up to 32 warps
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* slots, int& turn, int group) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
    }
    if (TPR > 32) {
        constexpr int WARPS = TPR / 32;
        float* set = slots + turn * (NORM_SLOTS / 2);
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) {
            const int warp = (threadIdx.x & (TPR - 1)) >> 5;
#pragma unroll
            for (int i = 0; i < N; ++i) set[i * 32 + warp] = v[i];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(TPR) : "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = set[i * 32];
#pragma unroll
            for (int k = 1; k < WARPS; ++k) s += set[i * 32 + k];
            v[i] = s;
        }
    }
}

// Mean (layer kind) and 1 / standard deviation of a row held in registers; v becomes the normed row.
template <int TPR, int V>
__device__ __forceinline__ void norm_row(float (&v)[NORM_VALUES], const NormParams& P, int lane, float* slots, int& turn, int group,
                                         float& mean, float& rstd) {
    mean = 0.0f;
    if (P.layer) {
        float s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) s[0] += v[j];              // columns past the row's end hold zeros
        row_sum<TPR, 1>(s, slots, turn, group);
        mean = s[0] / (float)P.dim;
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) v[j] = norm_column<TPR, V>(lane, j) < P.dim ? v[j] - mean : 0.0f;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NORM_VALUES; ++j) q[0] += v[j] * v[j];
    row_sum<TPR, 1>(q, slots, turn, group);
    rstd = 1.0f / sqrtf(q[0] / (float)P.dim + P.eps);
#pragma unroll
    for (int j = 0; j < NORM_VALUES; ++j) v[j] *= rstd;
}

// no y; y as it is; y through its own norm.  Backward: no y and no dr; y as it is, or no y but a dr (r is x, nothing is read of y); y through its own norm
enum NormMode : int { NORM_ONLY = 0, NORM_RESIDUAL = 1, NORM_POST = 2 };

RGB_HD constexpr int norm_cta(int tpr) { return tpr < 256 ? 256 : tpr; }

// One row from its values r (of x) and u (of y): r, h and the row's statistics.
template <int TPR, int V, int MODE>
__device__ __forceinline__ void norm_forward_row(const NormParams& P, int row, float (&r)[NORM_VALUES], float (&u)[NORM_VALUES], int lane, float* slots,
                                                 int& turn, int group, bool wide) {
    const size_t at = (size_t)row * P.dim;
    float t[NORM_VALUES], mean_y = 0.0f, rstd_y = 0.0f, mean, rstd;
    if (MODE != NORM_ONLY) {
        if (MODE == NORM_POST) {
            norm_row<TPR, V>(u, P, lane, slots, turn, group, mean_y, rstd_y);
            norm_load<TPR, V>(P.pw, P.dim, lane, wide, t);
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) u[j] *= t[j];
        }
        if (P.gate) {
            norm_load<TPR, V>(P.gate + (size_t)(row / P.group_rows) * P.dim, P.dim, lane, wide, t);
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) u[j] *= t[j];
        }
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) r[j] = P.scale * r[j] + u[j];
        norm_store<TPR, V>(P.r + at, P.dim, lane, wide, r);
    }
    norm_row<TPR, V>(r, P, lane, slots, turn, group, mean, rstd);
    norm_load<TPR, V>(P.w, P.dim, lane, wide, t);
#pragma unroll
    for (int j = 0; j < NORM_VALUES; ++j) r[j] *= t[j];
    if (P.b) {
        norm_load<TPR, V>(P.b, P.dim, lane, wide, t);
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) r[j] += t[j];
    }
    norm_store<TPR, V>(P.h + at, P.dim, lane, wide, r);
    if (P.stats && lane == 0) {
        P.stats[row] = mean;
        P.stats[(size_t)P.rows + row] = rstd;
        P.stats[2 * (size_t)P.rows + row] = mean_y;
        P.stats[3 * (size_t)P.rows + row] = rstd_y;
    }
}

// Forward: a row of threads for each row, the SM's other rows filling the pauses of its sums; or, where that leaves too little in flight,
// CTAs that stay and load their next row before they work on the present one.  That pays where few CTAs fit an SM (rows of 1024
// threads: 4096 x 8192 with post norm 109 us against 131, without 52 against 57) and for 64 and 128 threads without a block's output
// (65536 x 512: 48 us against 55; 43690 x 768: 54 against 65; 32768 x 1024: 48 against 55); elsewhere the registers of a second row cost more than they give (8192 x 4096:
// 134 us against 87 with post norm, 48 against 46 without; 16384 x 2048: 48 against 44; 131072 x 256: 47 against 44).
RGB_HD constexpr bool norm_stays(int tpr, int mode) { return tpr == 1024 || ((tpr == 64 || tpr == 128) && mode == NORM_ONLY); }

template <int TPR, int V, int MODE>
__global__ void __launch_bounds__(norm_cta(TPR))
block_norm_kernel(const NormParams P) {
    constexpr int GROUPS = norm_cta(TPR) / TPR;
    __shared__ float slots_all[GROUPS * NORM_SLOTS];
    const int group = threadIdx.x / TPR, lane = threadIdx.x & (TPR - 1);
    float* slots = slots_all + group * NORM_SLOTS;
    int turn = 0;
    const bool wide = P.wide != 0;
    long long row = (long long)blockIdx.x * GROUPS + group;
    if (row >= P.rows) return;                                           // whole warps, and whole rows of threads
    float x[NORM_VALUES], y[NORM_VALUES];
    norm_load<TPR, V>(P.x + (size_t)row * P.dim, P.dim, lane, wide, x);
    if (MODE != NORM_ONLY) norm_load<TPR, V>(P.y + (size_t)row * P.dim, P.dim, lane, wide, y);
    if constexpr (!norm_stays(TPR, MODE)) {
        norm_forward_row<TPR, V, MODE>(P, (int)row, x, y, lane, slots, turn, group, wide);
    } else {
        const long long step = (long long)gridDim.x * GROUPS;
        for (; row < P.rows; row += step) {
            float r[NORM_VALUES], u[NORM_VALUES];
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) {
                r[j] = x[j];
                if (MODE != NORM_ONLY) u[j] = y[j];
            }
            if (row + step < P.rows) {
                const size_t next = (size_t)(row + step) * P.dim;
                norm_load<TPR, V>(P.x + next, P.dim, lane, wide, x);
                if (MODE != NORM_ONLY) norm_load<TPR, V>(P.y + next, P.dim, lane, wide, y);
            }
            norm_forward_row<TPR, V, MODE>(P, (int)row, r, u, lane, slots, turn, group, wide);
        }
    }
}

// ------------------------------------------------------------------------------------------
// Backward: a row of threads walks over one range of rows (a part) and keeps its columns' sums in registers.
//
// Each row takes one or two sums over its threads, so plain loads would leave the memory system idle in between.  Every thread
// therefore copies the values that it will itself use of the next rows into shared memory asynchronously (cp.async; private
// slots, so no barrier guards them), NORM_STAGES rows ahead: 64 to 128 KB are in flight on an SM whatever the row is doing.
// 8192 x 4096 with post norm and gate: 132 us, 6.1 TB/s (226 us with plain loads).
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_4(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

RGB_HD constexpr int norm_stages(int tpr) { return tpr >= 1024 ? 1 : 2; }
RGB_HD constexpr int norm_tensors(int mode) { return mode == NORM_ONLY ? 2 : 4; }                // r, dh; dr, y
RGB_HD constexpr int norm_ring_bytes(int tpr, int mode) { return norm_stages(tpr) * norm_tensors(mode) * NORM_VALUES * 4 * norm_cta(tpr); }

// Slot of value j of this thread in a tensor's part of a stage, in floats: quads of a thread together, threads side by side.
template <int CTA, int V>
__device__ __forceinline__ int norm_slot(int j) { return V == 4 ? ((j >> 2) * CTA + (int)threadIdx.x) * 4 + (j & 3) : j * CTA + (int)threadIdx.x; }

template <int TPR, int V>
__device__ __forceinline__ void norm_fetch(uint32_t ring, const float* row, int dim, int lane, bool wide) {
    constexpr int CTA = norm_cta(TPR);
    if (V == 4 && wide) {
#pragma unroll
        for (int j = 0; j < NORM_VALUES; j += 4) {
            const int col = norm_column<TPR, V>(lane, j);
            copy_async_16(ring + 4 * norm_slot<CTA, V>(j), row + (col < dim ? col : 0), col < dim);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) {
            const int col = norm_column<TPR, V>(lane, j);
            copy_async_4(ring + 4 * norm_slot<CTA, V>(j), row + (col < dim ? col : 0), col < dim);
        }
    }
}
template <int TPR, int V>
__device__ __forceinline__ void norm_take(const float* ring, float (&v)[NORM_VALUES]) {
    constexpr int CTA = norm_cta(TPR);
    if (V == 4) {
#pragma unroll
        for (int j = 0; j < NORM_VALUES; j += 4) {
            const float4 q = *reinterpret_cast<const float4*>(ring + norm_slot<CTA, V>(j));
            v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) v[j] = ring[norm_slot<CTA, V>(j)];
    }
}

template <int TPR, int V, int MODE>
__global__ void __launch_bounds__(norm_cta(TPR), TPR < 512 ? 2 : 1)
block_norm_backward_kernel(const NormParams P) {
    constexpr int CTA = norm_cta(TPR), GROUPS = CTA / TPR, STAGES = norm_stages(TPR), TENSORS = norm_tensors(MODE);
    constexpr int TENSOR_FLOATS = NORM_VALUES * CTA, STAGE_FLOATS = TENSORS * TENSOR_FLOATS;
    extern __shared__ __align__(16) float ring[];
    __shared__ float slots_all[GROUPS * NORM_SLOTS];
    const int group = threadIdx.x / TPR, lane = threadIdx.x & (TPR - 1);
    float* slots = slots_all + group * NORM_SLOTS;
    int turn = 0;
    const int part = blockIdx.x * GROUPS + group;
    if (part >= P.parts_total) return;                                   // whole rows of threads; nothing below joins them
    const bool wide = P.wide != 0;
    const int gate_row = part / P.parts_per_group;
    const long long first = (long long)gate_row * P.group_rows + (long long)(part - gate_row * P.parts_per_group) * P.rows_per_part;
    const long long limit = (long long)(gate_row + 1) * P.group_rows;
    const int row_end = (int)(first + P.rows_per_part < limit ? first + P.rows_per_part : limit);
    const float inv_dim = 1.0f / (float)P.dim;
    const float* src_r = MODE == NORM_ONLY ? P.x : P.r;
    const bool use_y = MODE == NORM_POST || (MODE == NORM_RESIDUAL && P.gate);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);

    auto fetch = [&](int row) {
        if ((uint32_t)row < (uint32_t)row_end) {    // behind 2^31 - 1 rows the index has wrapped to a negative one
            const uint32_t at = ring_at + 4 * STAGE_FLOATS * (uint32_t)((row - (int)first) % STAGES);
            const size_t o = (size_t)row * P.dim;
            norm_fetch<TPR, V>(at, src_r + o, P.dim, lane, wide);
            norm_fetch<TPR, V>(at + 4 * TENSOR_FLOATS, P.dh + o, P.dim, lane, wide);
            if (MODE != NORM_ONLY) {
                if (P.dr) norm_fetch<TPR, V>(at + 8 * TENSOR_FLOATS, P.dr + o, P.dim, lane, wide);
                if (use_y) norm_fetch<TPR, V>(at + 12 * TENSOR_FLOATS, P.y + o, P.dim, lane, wide);
            }
        }
        copy_async_commit();                        // a group for every row, so that the count of groups in flight is fixed
    };
    float mean = 0.0f, rstd = 0.0f, mean_y = 0.0f, rstd_y = 0.0f;        // of the row to come
    auto fetch_stats = [&](int row) {
        if (row >= row_end) return;
        mean = P.stats[row];
        rstd = P.stats[(size_t)P.rows + row];
        if (MODE == NORM_POST) {
            mean_y = P.stats[2 * (size_t)P.rows + row];
            rstd_y = P.stats[3 * (size_t)P.rows + row];
        }
    };
#pragma unroll
    for (int s = 0; s < STAGES; ++s) fetch((int)first + s);
    fetch_stats((int)first);

    float w[NORM_VALUES], g[NORM_VALUES];
    float sum_w[NORM_VALUES] = {}, sum_b[NORM_VALUES] = {}, sum_q[NORM_VALUES] = {};
    norm_load<TPR, V>(P.w, P.dim, lane, wide, w);
    if (MODE != NORM_ONLY) {                        // gate times post weight: what D is multiplied by on its way to dy
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) g[j] = 1.0f;
        if (P.gate) norm_load<TPR, V>(P.gate + (size_t)gate_row * P.dim, P.dim, lane, wide, g);
        if (MODE == NORM_POST) {
            float t[NORM_VALUES];
            norm_load<TPR, V>(P.pw, P.dim, lane, wide, t);
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) g[j] *= t[j];
        }
    }
    for (int row = (int)first; row < row_end; ++row) {
        const size_t at = (size_t)row * P.dim;
        const float* stage = ring + (size_t)STAGE_FLOATS * ((row - (int)first) % STAGES);
        float r[NORM_VALUES], d[NORM_VALUES], dr[NORM_VALUES] = {}, y[NORM_VALUES] = {}, s[2] = {0.0f, 0.0f};
        copy_async_wait<STAGES - 1>();              // this row's group is complete
        norm_take<TPR, V>(stage, r);
        norm_take<TPR, V>(stage + TENSOR_FLOATS, d);
        if (MODE != NORM_ONLY) {
            if (P.dr) norm_take<TPR, V>(stage + 2 * TENSOR_FLOATS, dr);
            if (use_y) norm_take<TPR, V>(stage + 3 * TENSOR_FLOATS, y);
        }
        const float m_r = mean, s_r = rstd, m_y = mean_y, s_y = rstd_y;
        fetch((int)((uint32_t)row + STAGES));       // the slots just read
        fetch_stats(row + 1);
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) {
            r[j] = (r[j] - m_r) * s_r;              // past the row's end d is zero, which drops the value
            sum_w[j] += d[j] * r[j];
            sum_b[j] += d[j];
            d[j] *= w[j];
            s[0] += d[j] * r[j];
            s[1] += d[j];
        }
        row_sum<TPR, 2>(s, slots, turn, group);
        const float c1 = s[0] * inv_dim, c0 = P.layer ? s[1] * inv_dim : 0.0f;
#pragma unroll
        for (int j = 0; j < NORM_VALUES; ++j) {
            d[j] = dr[j] + s_r * (d[j] - r[j] * c1 - c0);
            r[j] = MODE == NORM_ONLY ? d[j] : P.scale * d[j];
        }
        if (P.dx) norm_store<TPR, V>(P.dx + at, P.dim, lane, wide, r);
        if (MODE == NORM_RESIDUAL) {
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) {
                sum_q[j] += d[j] * y[j];
                d[j] *= g[j];
            }
            if (P.dy) norm_store<TPR, V>(P.dy + at, P.dim, lane, wide, d);
        }
        if (MODE == NORM_POST) {
            float q[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) {
                const bool in = norm_column<TPR, V>(lane, j) < P.dim;
                y[j] = in ? (y[j] - m_y) * s_y : 0.0f;
                d[j] = in ? d[j] : 0.0f;
                sum_q[j] += d[j] * y[j];
                d[j] *= g[j];
                q[0] += d[j] * y[j];
                q[1] += d[j];
            }
            row_sum<TPR, 2>(q, slots, turn, group);
            const float e1 = q[0] * inv_dim, e0 = P.layer ? q[1] * inv_dim : 0.0f;
#pragma unroll
            for (int j = 0; j < NORM_VALUES; ++j) d[j] = s_y * (d[j] - y[j] * e1 - e0);
            if (P.dy) norm_store<TPR, V>(P.dy + at, P.dim, lane, wide, d);
        }
    }
    copy_async_wait<0>();
    float* out = P.parts + (size_t)part * 3 * P.dim;
    norm_store<TPR, V>(out, P.dim, lane, V == 4, sum_w);
    if (P.db) norm_store<TPR, V>(out + P.dim, P.dim, lane, V == 4, sum_b);
    if (P.dpw || P.dgate) norm_store<TPR, V>(out + 2 * (size_t)P.dim, P.dim, lane, V == 4, sum_q);
}

// Several gate rows: Q of each group from its parts, dgate, and g Q (the group's share of dpw) in place of the group's first Q.
static __global__ void __launch_bounds__(256)
norm_group_sums_kernel(const NormParams P) {
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= P.dim) return;
    for (int g = blockIdx.y; g < P.groups; g += gridDim.y) {
        float* first = P.parts + ((size_t)g * P.parts_per_group * 3 + 2) * P.dim + col;
        float q = 0.0f;
        for (int p = 0; p < P.parts_per_group; ++p) q += first[(size_t)p * 3 * P.dim];
        if (P.dgate) P.dgate[(size_t)g * P.dim + col] = P.pw ? P.pw[col] * q : q;
        if (P.parts_per_group > 0) *first = P.gate[(size_t)g * P.dim + col] * q;
    }
}

// Column sums of the parts: a CTA owns 32 columns, each of its 16 warps adds every sixteenth part in order, then the warps'
// sums are added in order.  blockIdx.y: 0 for dw, 1 for db, 2 for Q.
constexpr int NORM_SUM_WARPS = 16;
static __global__ void __launch_bounds__(32 * NORM_SUM_WARPS)
norm_column_sums_kernel(const NormParams P) {
    __shared__ float part[NORM_SUM_WARPS][32];
    const int which = blockIdx.y;
    if (which == 0 ? !P.dw : which == 1 ? !P.db : (!P.dpw && (!P.dgate || P.groups > 1))) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const bool by_group = which == 2 && P.groups > 1;
    const int items = by_group && P.parts_total > 0 ? P.groups : P.parts_total;     // no rows: no parts, zeros
    const size_t stride = (size_t)(by_group ? P.parts_per_group : 1) * 3 * P.dim;
    float s = 0.0f;
    if (col < P.dim) {
        const float* src = P.parts + (size_t)which * P.dim + col;
#pragma unroll 8
        for (int i = warp; i < items; i += NORM_SUM_WARPS) s += src[(size_t)i * stride];
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || col >= P.dim) return;
    for (int k = 1; k < NORM_SUM_WARPS; ++k) s += part[k][lane];
    if (which == 0) P.dw[col] = s;
    else if (which == 1) P.db[col] = s;
    else if (by_group) P.dpw[col] = s;
    else {
        if (P.dpw) P.dpw[col] = P.gate ? P.gate[col] * s : s;
        if (P.dgate) P.dgate[col] = P.pw ? P.pw[col] * s : s;
    }
}

}  // namespace rgb200
