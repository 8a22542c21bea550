// The product as a building block of other entry points of this library (defined in rgb200_api.cu).
#pragma once
#include <cuda_runtime.h>
#include "../../include/rgb200.h"

namespace rgb200 {

struct EpilogueParams;

// What the split of an operand does with infinities and NaN.  The plain products define their bits for finite values alone: a NaN is left out of
// its row's maximum, and the digits of either are whatever their bits give.  The operators of a training step must not turn them into
// finite losses and gradients.
enum NonFinite : int {
    NF_UNDEFINED = 0,   // the plain products
    NF_MARK = 1,        // a row that holds one is recorded with NONFINITE_EXPO: every output it takes part in is NaN
    NF_DROP = 2         // they do not count for the row's scale; for an operand whose partner holds zeros there (k-strided operands only)
};

// What gemm_with_epilogue may take as prepared in its workspace.
struct Prepared {
    // op(A)'s digit planes and exponents are in place: from a call with the same M, N, K, slices and transposition, or written
    // through plane_slots
    bool a = false;
    // op(B)'s are, from the previous call on this workspace with the same N, K, slices and transposition
    bool b = false;
    // Where the kernels report an expired wait, in place of the workspace's own word: an operation of several products keeps one
    // word, so that a later product does not clear an earlier one's report.  It is zeroed by the first call (zero_status, needs
    // both operands k-contiguous) or by the caller.
    int* status = nullptr;
    bool zero_status = false;
    // how this call splits op(A) and op(B), where it does
    NonFinite nonfinite_a = NF_MARK, nonfinite_b = NF_MARK;
};

// Where a product's workspace holds op(A): planes [slices][M][k_padded] and exponents [M].
struct PlaneSlots { signed char* planes; int* expo; int k_padded; };
cudaError_t plane_slots(int M, int N, int K, const rgb200_config& cfg, void* ws, PlaneSlots* out);

// C = epilogue(op(A) op(B)): rgb200_gemm_fp32_ws with an epilogue (EPI_*).  The workspace is the one rgb200_make_plan asks for.
// EPI_NONE is the plain product; the cross-entropy epilogues need the whole K in one pass (K within one INT32 accumulation).
// A may be null where it is prepared.
cudaError_t gemm_with_epilogue(const float* A, const float* B, float* C, int M, int N, int K, const rgb200_config& cfg, int epi,
                               const EpilogueParams& E, Prepared prepared, void* ws, size_t ws_bytes, cudaStream_t st);

// C [M, N] = A^T B over the rows of A [R, M] and B [R, N]: a weight's gradient.  One EPI_NONE product where the sums of R terms fit INT64; else
// (S = 3, more than 1 056 751 rows) one for each range of 2^20 rows, the later ones added in order.  `prepared` holds for one product only: a and b must
// be false for several.  Bytes of workspace, 0 where the sizes are not supported.
bool transposed_in_ranges(int R, int slices);
size_t transposed_product_bytes(int M, int N, int R, int slices);
cudaError_t transposed_product(const float* A, const float* B, float* C, int M, int N, int R, int slices, Prepared prepared, void* ws, size_t ws_bytes,
                               cudaStream_t st);

// Digit planes of src [R][C] (rows ld elements apart) as the row-scaled operand (k along the columns) and as the column-scaled one (k along the rows),
// from the bits of its rows' and columns' largest magnitudes (rgb200_dual.cuh).
cudaError_t launch_split_both(int slices, const float* src, int ld, int R, int C, const unsigned* row_max, const unsigned* col_max, const PlaneSlots& rows,
                              const PlaneSlots& cols, cudaStream_t st);

}  // namespace rgb200
