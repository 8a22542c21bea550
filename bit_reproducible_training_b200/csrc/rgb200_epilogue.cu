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
    kernel<<<grid, GEMM_THREADS, epilogue_smem<S>(), st>>>(a, b, P);
    return cudaGetLastError();
}

template <int EPI>
cudaError_t launch_slices(int S, int grid, const CUtensorMap& a, const CUtensorMap& b, const GemmParams& P, cudaStream_t st) {
    if (S == 1) return launch<1, EPI>(grid, a, b, P, st);
    if (S == 2) return launch<2, EPI>(grid, a, b, P, st);
    return launch<3, EPI>(grid, a, b, P, st);
}

// Row ranges of the backward pass, from the sizes alone: about six CTAs for each of the GPU's 148 SMs, at least 32 rows each.
int backward_ranges(int M, int N) {
    const int strips = (N + ACTB_COLS - 1) / ACTB_COLS;
    int ranges = (148 * 6 + strips - 1) / strips;
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
    return gemm_with_epilogue(A, B, C, M, N, K, *cfg, EPI_LINEAR, E, false, false, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" size_t rgb200_activation_backward_workspace(int M, int N) {
    if (M < 0 || N < 1) return 0;
    const size_t n = (size_t)backward_ranges(M, N) * N * sizeof(float);
    return n < 256 ? 256 : n;
}

extern "C" int rgb200_activation_backward(const float* dY, const float* Z, float* dZ, float* db, int M, int N, int activation, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    if (M < 0 || N < 1 || activation < 0 || activation >= ACT_COUNT || (!dZ && !db)) return cudaErrorInvalidValue;
    if (M > 0 && (!dY || (activation != ACT_NONE && !Z))) return cudaErrorInvalidValue;
    if (db && (!workspace || workspace_bytes < rgb200_activation_backward_workspace(M, N))) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess) return e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ranges = backward_ranges(M, N);
    ActBackwardParams P;
    P.dy = dY; P.z = Z; P.dz = dZ;
    P.parts = db ? static_cast<float*>(workspace) : nullptr;
    P.M = M; P.N = N; P.act = activation;
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    P.wide = aligned(dY) && aligned(Z) && aligned(dZ);
    if (M > 0) {
        P.rows_per_range = (M + ranges - 1) / ranges;
        const dim3 grid((N + ACTB_COLS - 1) / ACTB_COLS, (M + P.rows_per_range - 1) / P.rows_per_range);
        if (N % 4 == 0) activation_backward_kernel<4><<<grid, 32 * ACTB_WARPS, 0, st>>>(P);
        else activation_backward_kernel<1><<<grid, 32 * ACTB_WARPS, 0, st>>>(P);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        if (db) range_sums_kernel<<<(N + 31) / 32, 256, 0, st>>>(P.parts, (int)grid.y, N, db);
    } else if (db) {
        range_sums_kernel<<<(N + 31) / 32, 256, 0, st>>>(P.parts, 0, N, db);
    }
    return cudaGetLastError();
}
