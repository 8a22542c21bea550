// One matrix as the operand of two products: its digit planes with one scale per row, k running along the columns, and
// with one scale per column, k running along the rows.
//
// The gradient of a linear layer needs its dZ both ways (dX = dZ W, dW = dZ^T X), the cross entropy its piece of probabilities.
// Two pre-passes read the matrix once each and find the maxima themselves; here the kernel that produces the matrix has left
// the maxima of its rows and columns, and one read serves both.  Same exponents, same digits: the products' bits do not change.
// A maximum that is not finite marks its row or column (NF_MARK).
// Bound: HBM, (4 + 2 S) bytes a value; beside it about 45 instructions a value.  A CTA turns a 128 x 64 tile: eight 16-byte loads
// a thread, the row digits straight from the registers, then the tile through shared memory (quads exchanged by row, so that
// neither side meets bank conflicts) and 32 values of one column a thread, one 32-byte store a plane.
// S = 3, 8192 x 4096: 69 us = 4.9 TB/s; five CTAs an SM (48 registers) against four: 3 % faster, six: 15 % slower (spills).
#pragma once
#include "rgb200_prepass_cluster.cuh"

namespace rgb200 {

constexpr int DUAL_ROWS = 128, DUAL_COLS = 64, DUAL_THREADS = 256;
constexpr uint32_t INFINITY_BITS = 0x7F800000u;          // NaN counts as an infinity

struct DualParams {
    const float* src;               // [R][C], rows ld apart
    const uint32_t *row_max, *col_max;      // bits of the largest magnitudes (as integers: infinities and NaN lie above all others)
    int8_t *row_planes, *col_planes;        // [S][R][Cp], [S][C][Rp]
    int *row_expo, *col_expo;
    int R, C, ld, Rp, Cp;
};

template <int S>
__device__ __forceinline__ void dual_words(float a, float b, float c, float d, const QuantScale& q, bool plain, uint32_t (&w)[S]) {
    if (plain) quad_words<S, true>(a, b, c, d, q, 0.0f, w);
    else quad_words<S, false>(a, b, c, d, q, (float)q.lim, w);
}

// grid = (Cp / 64) * (Rp / 128), column tiles fastest
template <int S, bool VEC>
__global__ void __launch_bounds__(DUAL_THREADS, 5)
split_both_kernel(const DualParams P) {
    __shared__ __align__(16) float tile[DUAL_ROWS * DUAL_COLS];
    __shared__ int row_e[DUAL_ROWS], col_e[DUAL_COLS];
    const int t = threadIdx.x, quad = t & 15, sub = t >> 4;           // sixteen threads along a row of the tile
    const int col_tiles = P.Cp / DUAL_COLS, row_tile = blockIdx.x / col_tiles, col_tile = blockIdx.x - row_tile * col_tiles;
    const int r0 = row_tile * DUAL_ROWS, c0 = col_tile * DUAL_COLS;
    float4 v[8];
    const int col = c0 + quad * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = r0 + sub + 16 * i;
        const float* s = P.src + (size_t)row * P.ld + col;
        if (VEC) {                                       // ld is a multiple of four: the quad exists, its values behind column C do not count
            v[i] = row < P.R && col < P.C ? *reinterpret_cast<const float4*>(s) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
            const bool in = row < P.R;
            v[i] = make_float4(in && col < P.C ? s[0] : 0.f, in && col + 1 < P.C ? s[1] : 0.f, in && col + 2 < P.C ? s[2] : 0.f, in && col + 3 < P.C ? s[3] : 0.f);
        }
    }
    if (VEC && c0 + DUAL_COLS > P.C) {                    // the last tile of a row, one branch for the CTA
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i].y = col + 1 < P.C ? v[i].y : 0.f;
            v[i].z = col + 2 < P.C ? v[i].z : 0.f;
            v[i].w = col + 3 < P.C ? v[i].w : 0.f;
        }
    }
    if (t < DUAL_ROWS) {
        const int row = r0 + t;
        const int e = row < P.R ? scale_exponent(bits_f32(min(P.row_max[row], INFINITY_BITS))) : 0;
        row_e[t] = e;
        if (row < P.R && col_tile == 0) P.row_expo[row] = recorded_expo(e, true);
    } else if (t < DUAL_ROWS + DUAL_COLS) {
        const int j = t - DUAL_ROWS, c = c0 + j;
        const int e = c < P.C ? scale_exponent(bits_f32(min(P.col_max[c], INFINITY_BITS))) : 0;
        col_e[j] = e;
        if (c < P.C && row_tile == 0) P.col_expo[c] = recorded_expo(e, true);
    }
    __syncthreads();
    const size_t row_plane = (size_t)P.R * P.Cp, col_plane = (size_t)P.C * P.Rp;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int rr = sub + 16 * i, row = r0 + rr;
        *reinterpret_cast<float4*>(tile + (rr * 16 + (quad ^ (rr & 15))) * 4) = v[i];
        if (row < P.R) {
            const int e = row_e[rr];
            uint32_t w[S];
            dual_words<S>(v[i].x, v[i].y, v[i].z, v[i].w, quant_scale(e, S), plain_row(e), w);
#pragma unroll
            for (int p = 0; p < S; ++p) *reinterpret_cast<uint32_t*>(P.row_planes + p * row_plane + (size_t)row * P.Cp + col) = w[p];
        }
    }
    __syncthreads();
    // column j of the tile, 32 rows from 32 * (t / 64)
    const int j = t & 63, base = (t >> 6) * 32, c = c0 + j;
    if (c >= P.C) return;
    const int e = col_e[j];
    const QuantScale q = quant_scale(e, S);
    const bool plain = plain_row(e);
    uint32_t w[S][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rr = base + 4 * k + i;
            x[i] = tile[(rr * 16 + ((j >> 2) ^ (rr & 15))) * 4 + (j & 3)];
        }
        uint32_t o[S];
        dual_words<S>(x[0], x[1], x[2], x[3], q, plain, o);
#pragma unroll
        for (int p = 0; p < S; ++p) w[p][k] = o[p];
    }
#pragma unroll
    for (int p = 0; p < S; ++p)
        st_global_256(reinterpret_cast<uint32_t*>(P.col_planes + p * col_plane + (size_t)c * P.Rp + r0 + base), w[p][0], w[p][1], w[p][2], w[p][3], w[p][4],
                      w[p][5], w[p][6], w[p][7]);
}

}  // namespace rgb200
