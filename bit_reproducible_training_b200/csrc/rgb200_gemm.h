// The product as a building block of other entry points of this library (defined in rgb200_api.cu).
#pragma once
#include <cuda_runtime.h>
#include "../../include/rgb200.h"

namespace rgb200 {

struct EpilogueParams;

// C = epilogue(op(A) op(B)): rgb200_gemm_fp32_ws with an epilogue (EPI_*).  The workspace is the one rgb200_make_plan asks for.
// EPI_NONE is the plain product; the cross-entropy epilogues need the whole K in one pass (K within one INT32 accumulation).
// reuse_b: the workspace still holds B's digit planes from the previous call on it with the same N, K, slices and transposition;
// reuse_a: A's, from a call with the same M, N, K, slices, both operands k-contiguous (C = A B^T).
cudaError_t gemm_with_epilogue(const float* A, const float* B, float* C, int M, int N, int K, const rgb200_config& cfg, int epi,
                               const EpilogueParams& E, bool reuse_a, bool reuse_b, void* ws, size_t ws_bytes, cudaStream_t st);

}  // namespace rgb200
