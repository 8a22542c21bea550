// Launchers of the kernels with an epilogue (built in rgb200_epilogue.cu), called by the launch sequence in rgb200_api.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace rgb200 {

struct GemmParams;
struct EpilogueParams;
constexpr int EPI_TILE_N = 64;      // columns of C per tile in these kernels, whatever the slice count

// The general kernel over `tiles` tiles with epilogue `epi` (EPI_LINEAR and so on; P.epi holds its operands).
cudaError_t launch_gemm_epilogue(int slices, int epi, int grid, const CUtensorMap& a, const CUtensorMap& b, const GemmParams& P, cudaStream_t st);
// C = epilogue(round(sum of `parts` INT64 partials [parts][M][N])).
cudaError_t launch_round_epilogue(const long long* partial, int parts, const int* ea, const int* eb, int M, int N, float* C, int e0,
                                  const EpilogueParams& E, int sm_count, cudaStream_t st);

}  // namespace rgb200
