// Kernels with an epilogue and the entry point of its backward pass (include/rgb200_train.h).
#include <cstdint>
#include <mutex>

#include "../../include/rgb200_train.h"
#include "rgb200_host.h"
#include "rgb200_epilogue.h"
#include "rgb200_gemm.h"
#include "rgb200_epilogue.cuh"

namespace rgb200 {

static_assert(ACT_NONE == RGB200_ACT_NONE && ACT_RELU == RGB200_ACT_RELU && ACT_SILU == RGB200_ACT_SILU && ACT_GELU == RGB200_ACT_GELU &&
              ACT_GELU_TANH == RGB200_ACT_GELU_TANH, "activation codes");

namespace {

template <int S>
constexpr int epilogue_smem() { return GemmTraits<S, EPI_TILE_N>::SMEM_BYTES + 2 * EPI_WARPS * (EPI_TILE_N / 2) * 4; }

template <int S, int EPI>
cudaError_t launch(int grid, const CUtensorMap& a, const CUtensorMap& b, const GemmParams& P, cudaStream_t st) {
    auto kernel = gemm_i8_tcgen05_kernel<S, EPI_TILE_N, false, EPI>;
    static std::once_flag once[64];
    static cudaError_t err[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::call_once(once[dev], [&] { err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, epilogue_smem<S>()); });
    if (err[dev] != cudaSuccess) return err[dev];
    kernel<<<grid, gemm_threads(EPI), epilogue_smem<S>(), st>>>(a, b, P);
    return cudaGetLastError();
}

template <int EPI>
cudaError_t launch_slices(int S, int grid, const CUtensorMap& a, const CUtensorMap& b, const GemmParams& P, cudaStream_t st) {
    if (S == 1) return launch<1, EPI>(grid, a, b, P, st);
    if (S == 2) return launch<2, EPI>(grid, a, b, P, st);
    return launch<3, EPI>(grid, a, b, P, st);
}

// Row ranges of the backward pass, from the sizes alone: as many as give the 148 SMs two rounds of three CTAs each (what their registers
// hold) and not a few more, at least 32 rows each.  8192 x 4096 with gelu: 28 ranges (896 CTAs, a third round of eight) took 88 us, 27 take 75 us (5.4 TB/s).
constexpr int ACTB_MAX_SIZE = 0x7FFFFFFF - 4096;           // the kernel's indexes run up to a batch or a strip ahead, the ranges' arithmetic by their count
int backward_ranges(int M, int N) {
    const int strips = (N + ACTB_COLS - 1) / ACTB_COLS;
    int ranges = 148 * 6 / strips;
    if (ranges < 1) ranges = 1;
    if (ranges > (M + 31) / 32) ranges = (M + 31) / 32;
    if (ranges > 65535) ranges = 65535;
    return ranges;
}

}  // namespace

cudaError_t launch_gemm_epilogue(int slices, int epi, int grid, const CUtensorMap& a, const CUtensorMap& b, const GemmParams& P, cudaStream_t st) {
    if (epi == EPI_LINEAR) return launch_slices<EPI_LINEAR>(slices, grid, a, b, P, st);
    if (epi == EPI_LSE) return launch_slices<EPI_LSE>(slices, grid, a, b, P, st);
    if (epi == EPI_PROB) return launch_slices<EPI_PROB>(slices, grid, a, b, P, st);
    return cudaErrorInvalidValue;
}

cudaError_t launch_round_epilogue(const long long* partial, int parts, const int* ea, const int* eb, int M, int N, float* C, int e0,
                                  const EpilogueParams& E, int sm_count, cudaStream_t st) {
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = N % 4 == 0 && aligned(C) && aligned(E.residual) && aligned(E.pre);
    const size_t items = (size_t)M * N / (vec ? 4 : 1), want = (items + 255) / 256, cap = (size_t)sm_count * 32;
    const int blocks = (int)(want < cap ? want : cap);
    if (vec) round_partial_linear_kernel<true><<<blocks, 256, 0, st>>>(partial, parts, ea, eb, M, N, C, e0, E);
    else round_partial_linear_kernel<false><<<blocks, 256, 0, st>>>(partial, parts, ea, eb, M, N, C, e0, E);
    return cudaGetLastError();
}

}  // namespace rgb200

using namespace rgb200;

extern "C" int rgb200_gemm_epilogue_fp32_ws(const float* A, const float* B, float* C, int M, int N, int K, const rgb200_config* cfg,
                                            const rgb200_epilogue* epilogue, void* workspace, size_t workspace_bytes, void* stream) {
    if (!A || !B || !C || !cfg || !epilogue || epilogue->activation < 0 || epilogue->activation >= ACT_COUNT) return cudaErrorInvalidValue;
    EpilogueParams E = {};
    E.bias = epilogue->bias; E.residual = epilogue->residual; E.pre = epilogue->pre_activation; E.act = epilogue->activation;
    return gemm_with_epilogue(A, B, C, M, N, K, *cfg, EPI_LINEAR, E, Prepared(), workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" size_t rgb200_activation_backward_workspace(int M, int N) {
    if (M < 0 || M > ACTB_MAX_SIZE || N < 1 || N > ACTB_MAX_SIZE) return 0;
    const size_t n = (size_t)backward_ranges(M, N) * N * sizeof(float);
    return n < 256 ? 256 : n;
}

namespace {

// dZ (when P.dz), the columns' sums (db, with P.parts for the ranges') and, when P.row_max is set, dZ's maxima.
cudaError_t run_activation_backward(ActBackwardParams P, float* db, cudaStream_t st) {
    const int ranges = backward_ranges(P.M, P.N);
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    P.wide = aligned(P.dy) && aligned(P.z) && aligned(P.dz);
    dim3 grid((P.N + ACTB_COLS - 1) / ACTB_COLS, 0);
    if (P.M > 0) {
        P.rows_per_range = (P.M + ranges - 1) / ranges;
        grid.y = (P.M + P.rows_per_range - 1) / P.rows_per_range;
        if (P.N % 4 == 0) activation_backward_kernel<4><<<grid, 32 * ACTB_WARPS, 0, st>>>(P);
        else activation_backward_kernel<1><<<grid, 32 * ACTB_WARPS, 0, st>>>(P);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    if (db) range_sums_kernel<<<(P.N + 31) / 32, 256, 0, st>>>(P.parts, (int)grid.y, P.N, db);
    return cudaGetLastError();
}

constexpr size_t LB_ALIGN = 256;
size_t lb_round(size_t x) { return (x + LB_ALIGN - 1) / LB_ALIGN * LB_ALIGN; }

rgb200_config backward_config(int slices, bool ta) {
    rgb200_config c;
    rgb200_default_config(&c);
    c.slices = slices; c.trans_a = ta;
    return c;
}

// Workspace of the linear layer's backward pass: dZ (with an activation), its maxima, the ranges' column sums, and each product's own.
struct LinearBackwardLayout { size_t status, maxima, dz, parts, dx, dw, total, dx_bytes, dw_bytes; };
bool linear_backward_layout(int M, int N, int K, int act, int S, LinearBackwardLayout& L) {
    if (M < 1 || M > ACTB_MAX_SIZE || N < 1 || N > ACTB_MAX_SIZE || K < 1 || S < 1 || S > 3 || act < 0 || act >= ACT_COUNT) return false;
    const rgb200_config cx = backward_config(S, false);
    rgb200_layout_info ix;
    if (rgb200_layout(M, K, N, 1, &cx, &ix) != cudaSuccess) return false;
    L.dx_bytes = lb_round(ix.workspace_bytes);
    L.dw_bytes = lb_round(transposed_product_bytes(N, K, M, S));
    if (L.dw_bytes == 0) return false;
    L.status = 0;                            // one word, directly in front of the maxima: cleared together
    L.maxima = 4;
    L.dz = lb_round(L.maxima + (size_t)M * 4 + (size_t)N * 4);
    L.parts = L.dz + (act == ACT_NONE ? 0 : lb_round((size_t)M * N * 4));
    L.dx = L.parts + lb_round((size_t)backward_ranges(M, N) * N * 4);
    L.dw = L.dx + L.dx_bytes;
    L.total = L.dw + L.dw_bytes;
    return true;
}

}  // namespace

extern "C" int rgb200_activation_backward(const float* dY, const float* Z, float* dZ, float* db, int M, int N, int activation, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    if (M < 0 || M > ACTB_MAX_SIZE || N < 1 || N > ACTB_MAX_SIZE || activation < 0 || activation >= ACT_COUNT || (!dZ && !db)) return cudaErrorInvalidValue;
    if (M > 0 && (!dY || (activation != ACT_NONE && !Z))) return cudaErrorInvalidValue;
    if (db && (!workspace || workspace_bytes < rgb200_activation_backward_workspace(M, N))) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess) return e;
    ActBackwardParams P = {};
    P.dy = dY; P.z = Z; P.dz = dZ;
    P.parts = db ? static_cast<float*>(workspace) : nullptr;
    P.M = M; P.N = N; P.act = activation;
    return run_activation_backward(P, db, static_cast<cudaStream_t>(stream));
}

extern "C" size_t rgb200_linear_backward_workspace(int M, int N, int K, int activation, int slices) {
    LinearBackwardLayout L;
    return linear_backward_layout(M, N, K, activation, slices, L) ? L.total : 0;
}

extern "C" int rgb200_linear_backward(const float* dY, const float* Z, const float* X, const float* W, float* dX, float* dW, float* db, int M, int N, int K,
                                      int activation, int slices, void* workspace, size_t workspace_bytes, void* stream) {
    LinearBackwardLayout L;
    if (!linear_backward_layout(M, N, K, activation, slices, L) || !dY || (activation != ACT_NONE && !Z) || (!dX && !dW && !db)) return cudaErrorInvalidValue;
    if ((dX && !W) || (dW && !X)) return cudaErrorInvalidValue;
    if (!workspace || workspace_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & (LB_ALIGN - 1)) != 0) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess) return e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const bool both = dX && dW && !transposed_in_ranges(M, slices);
    ActBackwardParams P = {};
    P.dy = dY; P.z = Z;
    P.dz = activation != ACT_NONE && (dX || dW) ? reinterpret_cast<float*>(ws + L.dz) : nullptr;
    P.parts = db ? reinterpret_cast<float*>(ws + L.parts) : nullptr;
    P.M = M; P.N = N; P.act = activation;
    if (both) {
        P.row_max = reinterpret_cast<unsigned*>(ws + L.maxima);
        P.col_max = P.row_max + M;
    }
    if ((e = cudaMemsetAsync(ws + L.status, 0, L.maxima + (both ? (size_t)M * 4 + (size_t)N * 4 : 0), st)) != cudaSuccess) return e;
    if ((P.dz || db || both) && (e = run_activation_backward(P, db, st)) != cudaSuccess) return e;
    const float* dz = P.dz ? P.dz : dY;
    const rgb200_config cx = backward_config(slices, false);
    Prepared prepared;
    prepared.status = reinterpret_cast<int*>(ws + L.status);
    if (both) {
        PlaneSlots rows, cols;
        if ((e = plane_slots(M, K, N, cx, ws + L.dx, &rows)) != cudaSuccess || (e = plane_slots(N, K, M, backward_config(slices, true), ws + L.dw, &cols)) != cudaSuccess) return e;
        if ((e = launch_split_both(slices, dz, N, M, N, P.row_max, P.col_max, rows, cols, st)) != cudaSuccess) return e;
        prepared.a = true;
    }
    const EpilogueParams none = {};
    if (dX && (e = gemm_with_epilogue(dz, W, dX, M, K, N, cx, EPI_NONE, none, prepared, ws + L.dx, L.dx_bytes, st)) != cudaSuccess) return e;
    if (dW && (e = transposed_product(dz, X, dW, N, K, M, slices, prepared, ws + L.dw, L.dw_bytes, st)) != cudaSuccess) return e;
    return cudaSuccess;
}
