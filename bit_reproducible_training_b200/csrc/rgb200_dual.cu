// Launcher of the two-way split (rgb200_dual.cuh).
#include <cstdint>

#include "rgb200_gemm.h"
#include "rgb200_dual.cuh"

namespace rgb200 {

cudaError_t launch_split_both(int slices, const float* src, int ld, int R, int C, const unsigned* row_max, const unsigned* col_max, const PlaneSlots& rows,
                              const PlaneSlots& cols, cudaStream_t st) {
    DualParams P;
    P.src = src; P.row_max = row_max; P.col_max = col_max;
    P.row_planes = rows.planes; P.row_expo = rows.expo; P.Cp = rows.k_padded;
    P.col_planes = cols.planes; P.col_expo = cols.expo; P.Rp = cols.k_padded;
    P.R = R; P.C = C; P.ld = ld;
    const long long tiles = (long long)(P.Cp / DUAL_COLS) * (P.Rp / DUAL_ROWS);
    if (tiles > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)tiles;
    const bool vec = ld % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#define RGB_DUAL(S)                                                              \
    do {                                                                         \
        if (vec) split_both_kernel<S, true><<<grid, DUAL_THREADS, 0, st>>>(P);   \
        else split_both_kernel<S, false><<<grid, DUAL_THREADS, 0, st>>>(P);      \
    } while (0)
    if (slices == 1) RGB_DUAL(1);
    else if (slices == 2) RGB_DUAL(2);
    else RGB_DUAL(3);
#undef RGB_DUAL
    return cudaGetLastError();
}

}  // namespace rgb200
