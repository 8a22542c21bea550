// One AdamW step over many tensors in one launch, with first and second moments in FP32 or as 8-bit codes.
//
// The step is a fixed sequence of IEEE single operations per value (the library is built without FMA contraction), so its
// bits do not depend on how the values are spread over CTAs, launches or GPUs:
//   p1 = p * (1 - lr wd)
//   m' = m * b1 + g * (1 - b1)          v' = v * b2 + (g * g) * (1 - b2)
//   d  = sqrt(v') * (1 / sqrt(1 - b2^n)) + eps
//   p' = p1 - (m' / d) * (lr / (1 - b1^n))
// with every parenthesised constant formed in double precision and rounded once to FP32 (AdamwScalars).
//
// 8-bit states: blocks of 256 consecutive values of a tensor share one FP32 scale, the block's largest magnitude.
//   first moment   code q in [-127, 127]   value  ((q/127) |q/127|) * scale     q = RNE(127 sqrt(|m| / scale)) with m's sign
//   second moment  code q in [0, 255]      value  ((q/255)^2)^2 * scale         q = RNE(255 sqrt(sqrt(v / scale)))
// Companding by a square (a fourth power) spends the codes on small magnitudes: the relative step of m is 2/q, and sqrt(v),
// which is what the update divides by, has the same law as m.  A second moment that is not zero never gets the code
// zero, because the next step would divide by eps alone.  The update itself uses the moments before they are coded.
// A value that is not finite makes its block's scale NaN, so that the block reads as NaN (FP32 states keep a NaN too).
//
// Bound: HBM.  28 bytes a value in FP32 (p, m, v read and written, g read), 16 + 16/256 with 8-bit states.
// Measured, 124 M values in 111 tensors: FP32 states 511 us (6.8 TB/s, the copy rate); 8-bit states 451 us (4.5 TB/s), where the issue of
// about 90 instructions a value (the definition's root and quotient a third of them) takes longer than the memory: five CTAs an SM
// (48 registers) against four: 9 % faster, six: 2 % faster still with more spills; read-out of the values 226 us (5.5 TB/s).
// Split: a CTA takes a chunk of one tensor, found by bisection in the launch's table.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "rgb200_math.cuh"

namespace rgb200 {

constexpr int OPT_THREADS = 256;
constexpr int OPT_BLOCK = 256;          // values that share a scale
constexpr int OPT_MIN_CHUNK = 1024;     // values per CTA: a multiple of this
constexpr int OPT_SMALL_TABLE = 48, OPT_MEDIUM_TABLE = 160, OPT_LARGE_TABLE = 448;   // tensors a launch takes by value (448 x 60 bytes < 32 KB)

struct OptEntry {
    float* p;
    const float* g;
    void* m;               // float or int8 codes
    void* v;               // float or uint8 codes
    float* sm;             // scales (8-bit states)
    float* sv;
    long long n;
};

template <int CAP>
struct OptTable {
    OptEntry e[CAP];
    int first[CAP + 1];    // first chunk of each tensor; first[count] = number of chunks
    int count;
    int chunk;             // values per CTA
};

struct AdamwScalars { float decay, b1, c1, b2, c2, inv_sqrt_bc2, eps, step_size; };

// b^n by squaring, in double without contraction: the same bits on host and device.
RGB_HD double pow_int(double b, long long n) {
    double r = 1.0;
    for (; n > 0; n >>= 1) {
        if (n & 1) r = r * b;
        b = b * b;
    }
    return r;
}
RGB_HD AdamwScalars adamw_scalars(double lr, double b1, double b2, double eps, double wd, long long step) {
    AdamwScalars s;
    s.decay = (float)(1.0 - lr * wd);
    s.b1 = (float)b1; s.c1 = (float)(1.0 - b1);
    s.b2 = (float)b2; s.c2 = (float)(1.0 - b2);
    s.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow_int(b2, step)));
    s.eps = (float)eps;
    s.step_size = (float)(lr / (1.0 - pow_int(b1, step)));
    return s;
}

// Hyper-parameters of a launch: the scalars, or (step_word != null: steps counted on the device, for captured graphs)
// what they are formed from.
struct AdamwHyper {
    AdamwScalars s;
    double lr, b1, b2, eps, wd;
    const long long* step_word;
};

__device__ __forceinline__ void adamw_value(float& p, float g, float& m, float& v, const AdamwScalars& s) {
    const float p1 = __fmul_rn(p, s.decay);
    m = __fadd_rn(__fmul_rn(m, s.b1), __fmul_rn(g, s.c1));
    v = __fadd_rn(__fmul_rn(v, s.b2), __fmul_rn(__fmul_rn(g, g), s.c2));
    const float d = __fadd_rn(__fmul_rn(__fsqrt_rn(v), s.inv_sqrt_bc2), s.eps);
    p = __fsub_rn(p1, __fmul_rn(__fdiv_rn(m, d), s.step_size));
}

// Tensor that chunk `c` belongs to (first[] ascends; empty tensors own no chunk).
template <int CAP>
__device__ __forceinline__ int opt_find(const OptTable<CAP>& T, int c) {
    int lo = 0, hi = T.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (T.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ AdamwScalars adamw_load_scalars(const AdamwHyper& H, AdamwScalars* shared) {
    if (!H.step_word) return H.s;
    if (threadIdx.x == 0) *shared = adamw_scalars(H.lr, H.b1, H.b2, H.eps, H.wd, *H.step_word + 1);
    __syncthreads();
    return *shared;
}

__device__ __forceinline__ bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <int CAP>
__global__ void __launch_bounds__(OPT_THREADS)
adamw32_kernel(const __grid_constant__ OptTable<CAP> T, const __grid_constant__ AdamwHyper H) {
    __shared__ AdamwScalars shared;
    const AdamwScalars s = adamw_load_scalars(H, &shared);
    const int t = opt_find(T, blockIdx.x);
    const OptEntry& e = T.e[t];
    const long long at = (long long)((int)blockIdx.x - T.first[t]) * T.chunk;
    const int here = (int)(e.n - at < T.chunk ? e.n - at : T.chunk);
    float* p = e.p + at;
    const float* g = e.g + at;
    float* m = static_cast<float*>(e.m) + at;
    float* v = static_cast<float*>(e.v) + at;
    int done = 0;
    if (aligned_to(p, 16) && aligned_to(g, 16) && aligned_to(m, 16) && aligned_to(v, 16)) {
        const int quads = here >> 2;
        for (int i = threadIdx.x; i < quads; i += OPT_THREADS) {
            float4 pp = reinterpret_cast<const float4*>(p)[i], gg = reinterpret_cast<const float4*>(g)[i];
            float4 mm = reinterpret_cast<const float4*>(m)[i], vv = reinterpret_cast<const float4*>(v)[i];
            adamw_value(pp.x, gg.x, mm.x, vv.x, s);
            adamw_value(pp.y, gg.y, mm.y, vv.y, s);
            adamw_value(pp.z, gg.z, mm.z, vv.z, s);
            adamw_value(pp.w, gg.w, mm.w, vv.w, s);
            reinterpret_cast<float4*>(p)[i] = pp;
            reinterpret_cast<float4*>(m)[i] = mm;
            reinterpret_cast<float4*>(v)[i] = vv;
        }
        done = quads << 2;
    }
    for (int i = done + threadIdx.x; i < here; i += OPT_THREADS) {
        float pp = p[i], mm = m[i], vv = v[i];
        adamw_value(pp, g[i], mm, vv, s);
        p[i] = pp; m[i] = mm; v[i] = vv;
    }
}

// ------------------------------------------------------------------------------------------
// 8-bit codes.  A warp owns one block of 256 values, eight consecutive ones per lane.
// ------------------------------------------------------------------------------------------
constexpr float INV127 = (float)(1.0 / 127.0), INV255 = (float)(1.0 / 255.0);

// Conversions between codes and floats go through the mantissa of 2^23 + q and 1.5 * 2^23 + q (exact, and the addition
// rounds to nearest-even as the definition does): the conversion instructions share the slow pipe with the roots and reciprocals, of
// which a value needs five already.
constexpr float TWO23 = 8388608.0f, ROUNDER = 12582912.0f;
__device__ __forceinline__ float code_value(uint32_t word, int j, float offset) {      // float(byte j of word) - offset + 2^23
    return __fsub_rn(__uint_as_float(__byte_perm(word, 0x4B000000u, 0x7650u | j)), offset);
}
__device__ __forceinline__ float decode_m(uint32_t word, int j, float scale) {         // word: codes with their sign bits flipped
    const float t = __fmul_rn(code_value(word, j, TWO23 + 128.0f), INV127);
    return __fmul_rn(__fmul_rn(t, fabsf(t)), scale);
}
__device__ __forceinline__ float decode_v(uint32_t word, int j, float scale) {
    float t = __fmul_rn(code_value(word, j, TWO23), INV255);
    t = __fmul_rn(t, t);
    return __fmul_rn(__fmul_rn(t, t), scale);
}
// `scale`: the block's largest magnitude, or 1 for a block of zeros.  The definition's companded values, signed for m.
__device__ __forceinline__ float compand_m_exact(float m, float scale) {
    return copysignf(__fmul_rn(__fsqrt_rn(__fdiv_rn(fabsf(m), scale)), 127.0f), m);
}
__device__ __forceinline__ float compand_v_exact(float v, float scale) {
    return __fmul_rn(__fsqrt_rn(__fsqrt_rn(__fdiv_rn(v, scale))), 255.0f);
}
__device__ __forceinline__ float sqrt_fast(float x) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// The definition's quotient and roots, correctly rounded, would cost more time than the memory traffic.  `inv` = 1 / scale and the
// hardware's approximate root (relative error 2^-23) give nearly the same companded value: with u = 2^-24, |m| inv is off by 2 u,
// half of which the root keeps, 2 u for the root, u for the product, and the definition's own roundings are at most 2 u: 6 u of 127, below
// 4.6e-5; for v (two roots) 7 u of 255, below 1.1e-4.  A code can differ only where the value lies that close to a border between
// two codes; lanes that hold such a value redo it with the definition's operations.  inv = 0 marks a scale whose reciprocal
// leaves the normal range.
constexpr float BORDER_M = 0.5f - 6.0e-5f, BORDER_V = 0.5f - 1.4e-4f;
__device__ __forceinline__ float compand_m(float m, float inv) { return copysignf(sqrt_fast(fabsf(m) * inv) * 127.0f, m); }
__device__ __forceinline__ float compand_v(float v, float inv) { return sqrt_fast(sqrt_fast(v * inv)) * 255.0f; }
__device__ __forceinline__ float code_inverse(float scale) { return scale > 0x1p-100f && scale < 0x1p100f ? __frcp_rn(scale) : 0.0f; }
__device__ __forceinline__ float border_distance(float t) { return fabsf(t - ((t + ROUNDER) - ROUNDER)); }
__device__ __forceinline__ uint32_t code_bits(float t) { return __float_as_uint(t + ROUNDER); }   // the code in the low byte
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Largest magnitude over the warp's block, NaN if any value is not finite (the bits of non-negative floats order as
// integers, and infinity and NaN lie above every finite value).
template <bool SIGNED>
__device__ __forceinline__ float block_scale(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, SIGNED ? __float_as_uint(x[j]) & 0x7FFFFFFFu : __float_as_uint(x[j]));
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    return __uint_as_float(top >= 0x7F800000u ? 0x7FC00000u : top);
}

__device__ __forceinline__ void load8(const float* p, int live, bool wide, float (&x)[8]) {
    if (wide && live == 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = j < live ? p[j] : 0.0f;
    }
}
__device__ __forceinline__ void store8(float* p, int live, bool wide, const float (&x)[8]) {
    if (wide && live == 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < live) p[j] = x[j];
    }
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* q, int live, bool wide) {
    if (wide && live == 8) return *reinterpret_cast<const uint2*>(q);
    uint2 r = make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < live) (j < 4 ? r.x : r.y) |= (uint32_t)q[j] << (8 * (j & 3));
    return r;
}
__device__ __forceinline__ void store_codes(uint8_t* q, int live, bool wide, uint2 c) {
    if (wide && live == 8) { *reinterpret_cast<uint2*>(q) = c; return; }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < live) q[j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
}

__device__ __forceinline__ void decode_block(uint2 cm, uint2 cv, float sm, float sv, float (&m)[8], float (&v)[8]) {
    cm.x ^= 0x80808080u;
    cm.y ^= 0x80808080u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        m[j] = decode_m(j < 4 ? cm.x : cm.y, j & 3, sm);
        v[j] = decode_v(j < 4 ? cv.x : cv.y, j & 3, sv);
    }
}

__device__ __forceinline__ void encode_block(const float (&m)[8], const float (&v)[8], uint8_t* qm, uint8_t* qv, float* sm, float* sv,
                                             int lane, int live, bool wide) {
    const float tm = block_scale<true>(m), tv = block_scale<false>(v);
    const float dm = tm > 0.0f ? tm : 1.0f, dv = tv > 0.0f ? tv : 1.0f;      // NaN: 1, and the codes below are dropped
    const float im = code_inverse(dm), iv = code_inverse(dv);
    float x[8], y[8], worst = im == 0.0f || iv == 0.0f ? 1.0f : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = compand_m(m[j], im);
        y[j] = compand_v(v[j], iv);
        worst = fmaxf(worst, fmaxf(border_distance(x[j]) - (BORDER_M - BORDER_V), border_distance(y[j])));
    }
    if (worst >= BORDER_V) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (im == 0.0f || border_distance(x[j]) >= BORDER_M) x[j] = compand_m_exact(m[j], dm);
            if (iv == 0.0f || border_distance(y[j]) >= BORDER_V) y[j] = compand_v_exact(v[j], dv);
        }
    }
    uint32_t a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = code_bits(x[j]);
        b[j] = code_bits(v[j] > 0.0f ? fmaxf(y[j], 1.0f) : y[j]);            // a second moment that is not zero: at least code 1
    }
    uint2 cm = make_uint2(pack4(a[0], a[1], a[2], a[3]), pack4(a[4], a[5], a[6], a[7]));
    uint2 cv = make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
    if (isnan(tm)) cm = make_uint2(0u, 0u);
    if (isnan(tv)) cv = make_uint2(0u, 0u);
    store_codes(qm, live, wide, cm);
    store_codes(qv, live, wide, cv);
    if (lane == 0) { *sm = tm; *sv = tv; }
}

enum OptMode : int { OPT_STEP, OPT_READ, OPT_WRITE };   // update; codes -> values; values -> codes

template <OptMode MODE, bool FULL>
__device__ __forceinline__ void opt_block(const OptEntry& e, const AdamwScalars& s, long long block_at, long long at, int lane, bool any_wide) {
    const bool wide = FULL || any_wide;
    const int live = FULL ? 8 : at >= e.n ? 0 : (e.n - at < 8 ? (int)(e.n - at) : 8);
    float* sm = e.sm + block_at / OPT_BLOCK;
    float* sv = e.sv + block_at / OPT_BLOCK;
    uint8_t* qm = static_cast<uint8_t*>(e.m) + at;
    uint8_t* qv = static_cast<uint8_t*>(e.v) + at;
    float m[8], v[8];
    if (MODE != OPT_WRITE) decode_block(load_codes(qm, live, wide), load_codes(qv, live, wide), *sm, *sv, m, v);
    if (MODE == OPT_STEP) {
        float p[8], g[8];
        load8(e.p + at, live, wide, p);
        load8(e.g + at, live, wide, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            adamw_value(p[j], g[j], m[j], v[j], s);
            if (j >= live) m[j] = v[j] = 0.0f;                          // lanes past the tensor's end do not set its scale
        }
        store8(e.p + at, live, wide, p);
    } else if (MODE == OPT_READ) {
        store8(e.p + at, live, wide, m);
        store8(const_cast<float*>(e.g) + at, live, wide, v);
    } else {
        load8(e.p + at, live, wide, m);
        load8(e.g + at, live, wide, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += 0.0f;                       // -0 is a zero, and its bits are not below all others' (block_scale)
    }
    if (MODE != OPT_READ) encode_block(m, v, qm, qv, sm, sv, lane, live, wide);
}

// OPT_STEP: p, g and the codes.  OPT_READ: the moments' values go to p (first) and g (second, written through a cast
// away of const by the host's table); OPT_WRITE: they come from there.
template <int CAP, OptMode MODE>
__global__ void __launch_bounds__(OPT_THREADS, 5)
adamw8_kernel(const __grid_constant__ OptTable<CAP> T, const __grid_constant__ AdamwHyper H) {
    __shared__ AdamwScalars shared;
    AdamwScalars s = {};
    if (MODE == OPT_STEP) s = adamw_load_scalars(H, &shared);
    const int t = opt_find(T, blockIdx.x);
    const OptEntry& e = T.e[t];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long chunk_at = (long long)((int)blockIdx.x - T.first[t]) * T.chunk;
    const bool wide = aligned_to(e.p, 16) && aligned_to(e.g, 16) && aligned_to(e.m, 8) && aligned_to(e.v, 8);
    for (int b = warp; b < T.chunk / OPT_BLOCK; b += OPT_THREADS / 32) {
        const long long block_at = chunk_at + (long long)b * OPT_BLOCK;
        if (block_at >= e.n) break;                                     // uniform over the warp
        const long long at = block_at + lane * 8;
        // whole blocks of aligned tensors go without the checks that ragged ends and odd addresses need
        if (wide && e.n - block_at >= OPT_BLOCK) opt_block<MODE, true>(e, s, block_at, at, lane, true);
        else opt_block<MODE, false>(e, s, block_at, at, lane, wide);
    }
}

static __global__ void advance_step_kernel(long long* step_word) { *step_word += 1; }

}  // namespace rgb200
