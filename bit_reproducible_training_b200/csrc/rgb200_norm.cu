// Host side of the block-norm entry points declared in include/rgb200_train.h.
#include <mutex>

#include "../../include/rgb200_train.h"
#include "rgb200_host.h"
#include "rgb200_norm.cuh"

namespace rgb200 {
namespace {

// Threads of a row, from its length alone.
int norm_threads(int dim) {
    int t = 32;
    while (t * NORM_VALUES < dim) t *= 2;
    return t;
}

bool good_norm(const rgb200_block_norm* n) {
    if (!n || n->rows < 0 || n->dim < 1 || n->dim > NORM_MAX_DIM || n->groups < 1 || (n->kind != RGB200_NORM_RMS && n->kind != RGB200_NORM_LAYER)) return false;
    if (!(n->eps >= 0.0f) || n->scale != n->scale) return false;
    if (n->rows % n->groups != 0 || n->groups > NORM_MAX_GROUPS) return false;
    if (!n->gate && n->groups != 1) return false;
    if (n->rows > 0 && (!n->x || !n->weight || (!n->y && (n->post_weight || n->gate)))) return false;    // no rows: no tensors needed
    return true;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Row ranges of the backward pass, from the sizes alone: as many as fill the GPU's 148 SMs with 512 threads each (or one row
// of 1024), at least eight rows long so that their column sums stay a small part of the traffic.
struct NormParts { int per_group, rows, total; };
NormParts norm_parts(int rows, int dim, int groups) {
    NormParts p = {0, 0, 0};
    if (rows == 0) return p;
    const int group_rows = rows / groups, tpr = norm_threads(dim);
    long long want = 148ll * (tpr <= 512 ? 512 / tpr : 1) / groups;
    if (want < 1) want = 1;
    if (want > (group_rows - 1) / 8 + 1) want = (group_rows - 1) / 8 + 1;
    p.rows = (int)((group_rows - 1) / want + 1);               // group_rows may be 2^31 - 1
    p.per_group = (group_rows - 1) / p.rows + 1;
    p.total = p.per_group * groups;
    return p;
}

NormParams norm_params(const rgb200_block_norm* n) {
    NormParams P = {};
    P.x = n->x; P.y = n->y; P.w = n->weight; P.b = n->bias; P.pw = n->post_weight; P.gate = n->gate;
    P.r = n->r; P.h = n->h; P.stats = n->stats;
    P.rows = n->rows; P.dim = n->dim; P.groups = n->groups;
    P.group_rows = n->rows > 0 ? n->rows / n->groups : 1;
    P.layer = n->kind == RGB200_NORM_LAYER; P.scale = n->scale; P.eps = n->eps;
    P.dr = n->dr; P.dh = n->dh; P.dx = n->dx; P.dy = n->dy;
    P.dw = n->dweight; P.db = n->dbias; P.dpw = n->dpost_weight; P.dgate = n->dgate;
    P.wide = n->dim % 4 == 0;
    for (const void* p : {(const void*)n->x, (const void*)n->y, (const void*)n->weight, (const void*)n->bias, (const void*)n->post_weight, (const void*)n->gate,
                          (const void*)n->r, (const void*)n->h, (const void*)n->dr, (const void*)n->dh, (const void*)n->dx, (const void*)n->dy})
        if (!aligned16(p)) P.wide = 0;
    return P;
}

template <int TPR, int V, int MODE>
cudaError_t launch_backward(const NormParams& P, int grid, cudaStream_t st) {
    auto kernel = block_norm_backward_kernel<TPR, V, MODE>;
    constexpr int BYTES = norm_ring_bytes(TPR, MODE);
    static std::once_flag once[64];
    static cudaError_t err[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::call_once(once[dev], [&] { err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES); });
    if (err[dev] != cudaSuccess) return err[dev];
    kernel<<<grid, norm_cta(TPR), BYTES, st>>>(P);
    return cudaGetLastError();
}

template <int TPR, int V>
cudaError_t launch_norm(const NormParams& P, bool backward, cudaStream_t st) {
    constexpr int CTA = norm_cta(TPR), GROUPS = CTA / TPR;
    const int items = backward ? P.parts_total : P.rows;
    int grid = (items - 1) / GROUPS + 1;
    if (!backward) {
        const int mode = !P.y ? NORM_ONLY : !P.pw ? NORM_RESIDUAL : NORM_POST, resident = 148 * (2048 / CTA);
        if (norm_stays(TPR, mode) && grid > resident) grid = resident;
        if (!P.y) block_norm_kernel<TPR, V, NORM_ONLY><<<grid, CTA, 0, st>>>(P);
        else if (!P.pw) block_norm_kernel<TPR, V, NORM_RESIDUAL><<<grid, CTA, 0, st>>>(P);
        else block_norm_kernel<TPR, V, NORM_POST><<<grid, CTA, 0, st>>>(P);
        return cudaGetLastError();
    }
    if (!P.y && !P.dr) return launch_backward<TPR, V, NORM_ONLY>(P, grid, st);
    if (!P.pw) return launch_backward<TPR, V, NORM_RESIDUAL>(P, grid, st);
    return launch_backward<TPR, V, NORM_POST>(P, grid, st);
}

template <int V>
cudaError_t dispatch_norm(const NormParams& P, bool backward, cudaStream_t st) {
    switch (norm_threads(P.dim)) {
        case 32: return launch_norm<32, V>(P, backward, st);
        case 64: return launch_norm<64, V>(P, backward, st);
        case 128: return launch_norm<128, V>(P, backward, st);
        case 256: return launch_norm<256, V>(P, backward, st);
        case 512: return launch_norm<512, V>(P, backward, st);
        default: return launch_norm<1024, V>(P, backward, st);
    }
}

}  // namespace
}  // namespace rgb200

using namespace rgb200;

extern "C" int rgb200_block_norm_forward(const rgb200_block_norm* n, void* stream) {
    if (!good_norm(n)) return cudaErrorInvalidValue;
    if (n->rows > 0 && (!n->h || (n->y && !n->r))) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess || n->rows == 0) return e;
    const NormParams P = norm_params(n);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return P.dim % 4 == 0 ? dispatch_norm<4>(P, false, st) : dispatch_norm<1>(P, false, st);
}

extern "C" size_t rgb200_block_norm_backward_workspace(int rows, int dim, int groups) {
    if (rows < 0 || dim < 1 || dim > NORM_MAX_DIM || groups < 1 || groups > NORM_MAX_GROUPS || rows % groups != 0) return 0;
    const size_t n = (size_t)norm_parts(rows, dim, groups).total * 3 * dim * sizeof(float);
    return n < 256 ? 256 : n;
}

extern "C" int rgb200_block_norm_backward(const rgb200_block_norm* n, void* workspace, size_t workspace_bytes, void* stream) {
    if (!good_norm(n) || !workspace || workspace_bytes < rgb200_block_norm_backward_workspace(n->rows, n->dim, n->groups) || !aligned16(workspace))
        return cudaErrorInvalidValue;
    if (n->rows > 0 && (!n->dh || !n->stats || (n->y && !n->r))) return cudaErrorInvalidValue;
    if ((n->dy && !n->y) || (n->dpost_weight && !n->post_weight) || (n->dgate && !n->gate)) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess) return e;
    NormParams P = norm_params(n);
    const NormParts parts = norm_parts(n->rows, n->dim, n->groups);
    P.parts = static_cast<float*>(workspace);
    P.rows_per_part = parts.rows; P.parts_per_group = parts.per_group; P.parts_total = parts.total;
    if (!P.y) {                              // r is x itself, with a weight of one in the stream's gradient
        P.r = const_cast<float*>(P.x);       // only read
        P.scale = 1.0f;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n->rows > 0) {
        e = P.dim % 4 == 0 ? dispatch_norm<4>(P, true, st) : dispatch_norm<1>(P, true, st);
        if (e != cudaSuccess) return e;
    }
    if (P.dgate || P.dpw) {
        if (P.groups > 1)
            norm_group_sums_kernel<<<dim3((P.dim + 255) / 256, P.groups < 4096 ? P.groups : 4096), 256, 0, st>>>(P);
    }
    if (P.dw || P.db || P.dpw || P.dgate)
        norm_column_sums_kernel<<<dim3((P.dim + 31) / 32, P.dgate || P.dpw ? 3 : 2), 32 * NORM_SUM_WARPS, 0, st>>>(P);
    return cudaGetLastError();
}
