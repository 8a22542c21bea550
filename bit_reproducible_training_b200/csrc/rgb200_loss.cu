// Cross entropy of logits X W^T against targets in pieces of the vocabulary, without the logits (include/rgb200_train.h).
//
// Forward, for each piece of words: the product X W_piece^T runs with an epilogue that keeps, of each row and each 32 columns, the
// maximum and the sum of exponentials without the target's (8 bytes instead of 128), and the target's logit; a small kernel joins them into the
// rows' running statistics.  Backward, for each piece: the product again, now leaving P = g softmax without the targets' own
// entries in FP32 (one piece at a time), then dX += P W_piece (the running dX is the epilogue's residual) and
// dW_piece = P^T X.  The targets' entries (p - 1) g are kept apart: beside them the rest of a row is small, and in one matrix
// with them it would lose its low digits to their scale.  They enter as dX's start and as additions to dW at the end.
//
// Work: 4 products of 2 N V D operations (one more than with stored logits), each at the rate of the library's products; what is
// moved beside them is a few passes over one piece of P.
// Measured, 8192 x 50257 x 768: 9.28 ms of kernels, of them the statistics' product 2.05, the probabilities' 2.19 (both at K = 768, where
// the tensor pipe is 67 % busy), dX 1.91, dW 1.72, the two-way split of P 0.92, the splits of X and W 0.33, the rest 0.15.
#include <cstdint>

#include "../../include/rgb200_train.h"
#include "rgb200_epilogue.h"
#include "rgb200_gemm.h"
#include "rgb200_host.h"
#include "rgb200_loss.cuh"
#include "rgb200_mma.cuh"

namespace rgb200 {
namespace {

constexpr size_t XENT_ALIGN = 256;
size_t round_up(size_t x) { return (x + XENT_ALIGN - 1) / XENT_ALIGN * XENT_ALIGN; }

rgb200_config product_config(int slices, bool ta, bool tb) {
    rgb200_config c;
    rgb200_default_config(&c);
    c.slices = slices; c.trans_a = ta; c.trans_b = tb;
    return c;
}

bool product_bytes(int M, int N, int K, int slices, bool ta, bool tb, size_t* bytes) {
    const rgb200_config c = product_config(slices, ta, tb);
    rgb200_layout_info info;
    if (rgb200_layout(M, N, K, 1, &c, &info) != cudaSuccess) return false;
    *bytes = round_up(info.workspace_bytes);
    return true;
}

// Words per piece: near-equal multiples of 64 no wider than `limit`.
int piece_words(int vocab, int limit) {
    const int pieces = (vocab + limit - 1) / limit;
    const int w = ((vocab + pieces - 1) / pieces + 63) / 64 * 64;
    return w < vocab ? w : vocab;
}
// Few launches and bounded buffers: a piece's digit planes of W stay near 100 MB a copy (2^25 values), the forward pass's statistics below
// 64 MB (2^28 values of logits).
int bounded_words(long long most, int dim) {
    long long w = (1ll << 25) / dim;
    if (w > most) w = most;
    if (w > 65536) w = 65536;
    return w < 1024 ? 1024 : (int)(w / 128 * 128);
}
int forward_words(int rows, int vocab, int dim) { return piece_words(vocab, bounded_words((1ll << 28) / rows, dim)); }
// Words per piece of the backward pass, a multiple of 128 (or the whole vocabulary).  P of one piece holds at most 2^25 values, or up to
// 2^26 in pieces of up to 8192 words, while pieces of 1024 words allow it; below that the width is the one whose products fill the
// SMs' rounds best.  Cost in k blocks of one SM's tensor pipe: rounds of tiles times k blocks for the three products, and for each
// piece the time of its other kernels (about 30 us, 85 blocks).  8 rows of 256 against 50000 words: 568 us in pieces of at most
// 8192 words, most of it launches, 251 us in one.
int backward_words(int rows, int vocab, int dim) {
    long long most = (1ll << 26) / rows;
    if (most > 8192) most = (1ll << 25) / rows > 8192 ? (1ll << 25) / rows : 8192;
    const int limit = bounded_words(most, dim);
    if (vocab <= limit) return vocab;
    auto up = [](long long a, long long b) { return (a + b - 1) / b; };
    const long long row_tiles = up(rows, 128), dim_tiles = up(dim, EPI_TILE_N), row_blocks = up(rows, 128), dim_blocks = up(dim, 128);
    auto cost = [&](long long words) {
        return up(row_tiles * up(words, EPI_TILE_N), 148) * dim_blocks + up(row_tiles * dim_tiles, 148) * up(words, 128) +
               up(up(words, 128) * dim_tiles, 148) * row_blocks + 85;
    };
    int best = limit;
    long long best_cost = -1;
    for (int w = limit; w >= limit / 2 && w >= 1024; w -= 128) {
        const long long pieces = vocab / w, rest = vocab % w, c = pieces * cost(w) + (rest ? cost(rest) : 0);
        if (best_cost < 0 || c < best_cost) { best = w; best_cost = c; }
    }
    return best;
}

// Row length of P when one split takes it both ways: whole tiles of the product, so that an odd vocabulary does not leave its rows at odd
// addresses (1000 x 32003 x 512: the product's kernel takes 134 us against 264 with rows of 32003).
int padded_words(int words) { return (words + EPI_TILE_N - 1) / EPI_TILE_N * EPI_TILE_N; }

struct ForwardLayout { int words; size_t status, product, product_bytes, parts, running, total; };
bool forward_layout(int N, int V, int D, int S, ForwardLayout& L) {
    L.words = forward_words(N, V, D);
    size_t bytes;
    if (!product_bytes(N, L.words, D, S, false, true, &bytes)) return false;
    L.status = 0;
    L.product = XENT_ALIGN;
    L.product_bytes = bytes;
    L.parts = L.product + bytes;
    L.running = L.parts + round_up((size_t)2 * ((L.words + EPI_TILE_N - 1) / EPI_TILE_N) * N * sizeof(float2));
    L.total = L.running + round_up((size_t)N * sizeof(float2));
    return true;
}

struct BackwardLayout { int words; size_t status, listed, maxima, weight, coefficient, list, first, not_last, p, logits, dx, dw, total, logits_bytes, dx_bytes, dw_bytes; };
bool backward_layout(int N, int V, int D, int S, BackwardLayout& L) {
    L.words = backward_words(N, V, D);
    if (!product_bytes(N, L.words, D, S, false, true, &L.logits_bytes) || !product_bytes(N, D, L.words, S, false, false, &L.dx_bytes) ||
        (L.dw_bytes = round_up(transposed_product_bytes(L.words, D, N, S))) == 0)
        return false;
    // the last piece may be narrower, and a narrower product can be planned with more K ranges
    const int rest = V - (V - 1) / L.words * L.words;
    size_t b;
    if (!product_bytes(N, D, rest, S, false, false, &b)) return false;
    if (b > L.dx_bytes) L.dx_bytes = b;
    if ((b = round_up(transposed_product_bytes(rest, D, N, S))) == 0) return false;
    if (b > L.dw_bytes) L.dw_bytes = b;
    L.status = 0;                            // status, listed and the first piece's maxima are cleared together
    L.listed = 4;
    L.maxima = 8;
    L.weight = round_up(L.maxima + (size_t)N * 4 + (size_t)L.words * 4);
    L.coefficient = L.weight + round_up((size_t)N * 4);
    L.list = L.coefficient + round_up((size_t)N * 4);
    L.first = L.list + round_up((size_t)N * 4);
    L.not_last = L.first + (size_t)V * 4;
    L.p = L.first + round_up((size_t)V * 8);
    L.logits = L.p + round_up((size_t)N * padded_words(L.words) * 4);
    L.dx = L.logits + L.logits_bytes;
    L.dw = L.dx + L.dx_bytes;
    L.total = L.dw + L.dw_bytes;
    return true;
}

bool good_sizes(int N, int V, int D, int S) {
    return N >= 1 && N <= (1 << 30) && V >= 1 && V <= (1 << 30) && D >= 1 && S >= 1 && S <= 3 && D <= max_k_per_pass(S) / BLOCK_K * BLOCK_K;
}

}  // namespace
}  // namespace rgb200

using namespace rgb200;

extern "C" size_t rgb200_linear_xent_workspace(int N, int V, int D, int slices, int backward) {
    if (!good_sizes(N, V, D, slices)) return 0;
    ForwardLayout F;
    BackwardLayout B;
    if (backward) return backward_layout(N, V, D, slices, B) ? B.total : 0;
    return forward_layout(N, V, D, slices, F) ? F.total : 0;
}

extern "C" int rgb200_linear_xent_forward(const float* X, const float* W, const long long* target, long long ignore_index, int reduction, int N, int V,
                                          int D, int slices, float* loss, float* nll, float* lse, float* target_rest, float* inv_count,
                                          void* workspace, size_t workspace_bytes, void* stream) {
    if (!good_sizes(N, V, D, slices) || !X || !W || !target || !nll || !lse || !target_rest || !workspace) return cudaErrorInvalidValue;
    if (reduction < RGB200_REDUCE_NONE || reduction > RGB200_REDUCE_SUM || (reduction != RGB200_REDUCE_NONE && (!loss || !inv_count))) return cudaErrorInvalidValue;
    ForwardLayout L;
    if (!forward_layout(N, V, D, slices, L)) return cudaErrorInvalidValue;
    if (workspace_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & (XENT_ALIGN - 1)) != 0) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess) return e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const rgb200_config cfg = product_config(slices, false, true);
    EpilogueParams E = {};
    E.target = target;
    E.lse_parts = reinterpret_cast<float2*>(ws + L.parts);
    E.target_logit = target_rest;            // the logits, until the last join leaves the others' probability in their place
    for (int at = 0; at < V; at += L.words) {
        const int words = V - at < L.words ? V - at : L.words;
        E.first_word = at;
        // C is not written; the product's other operand checks want an address
        if ((e = gemm_with_epilogue(X, W + (size_t)at * D, nll, N, words, D, cfg, EPI_LSE, E,
                                    Prepared{at > 0 && words == L.words, false, reinterpret_cast<int*>(ws + L.status), at == 0}, ws + L.product,
                                    L.product_bytes, st)) != cudaSuccess)
            return e;
        // the last half tile of a piece has a part only if it has columns
        const int parts = (words + EPI_TILE_N / 2 - 1) / (EPI_TILE_N / 2);
        xent_join_kernel<<<(N + XENT_ROWS - 1) / XENT_ROWS, 32 * XENT_WARPS, 0, st>>>(
            E.lse_parts, parts, reinterpret_cast<float2*>(ws + L.running), N, at == 0, at + words == V, target, ignore_index, V, target_rest, lse, nll);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    if (reduction != RGB200_REDUCE_NONE)
        xent_reduce_kernel<<<1, 1024, 0, st>>>(nll, target, ignore_index, N, reduction == RGB200_REDUCE_MEAN, loss, inv_count);
    return cudaGetLastError();
}

extern "C" int rgb200_linear_xent_backward(const float* X, const float* W, const long long* target, long long ignore_index, int reduction, int N, int V,
                                           int D, int slices, const float* lse, const float* target_rest, const float* inv_count, const float* dloss,
                                           float* dX, float* dW, void* workspace, size_t workspace_bytes, void* stream) {
    if (!good_sizes(N, V, D, slices) || !X || !W || !target || !lse || !target_rest || !dloss || (!dX && !dW) || !workspace) return cudaErrorInvalidValue;
    if (reduction < RGB200_REDUCE_NONE || reduction > RGB200_REDUCE_SUM || (reduction != RGB200_REDUCE_NONE && !inv_count)) return cudaErrorInvalidValue;
    BackwardLayout L;
    if (!backward_layout(N, V, D, slices, L)) return cudaErrorInvalidValue;
    if (workspace_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & (XENT_ALIGN - 1)) != 0) return cudaErrorInvalidValue;
    cudaError_t e = check_b200();
    if (e != cudaSuccess) return e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    float* weight = reinterpret_cast<float*>(ws + L.weight);
    float* coefficient = reinterpret_cast<float*>(ws + L.coefficient);
    int* list = reinterpret_cast<int*>(ws + L.list);
    int* listed = reinterpret_cast<int*>(ws + L.listed);
    int* first = reinterpret_cast<int*>(ws + L.first);
    int* not_last = reinterpret_cast<int*>(ws + L.not_last);
    const bool both = dX && dW && !transposed_in_ranges(N, slices);
    const size_t maxima_bytes = (size_t)N * 4 + (size_t)L.words * 4;
    float* P = reinterpret_cast<float*>(ws + L.p);

    if ((e = cudaMemsetAsync(ws, 0, L.maxima + (both ? maxima_bytes : 0), st)) != cudaSuccess) return e;
    if ((e = cudaMemsetAsync(first, 0x7F, (size_t)V * 8, st)) != cudaSuccess) return e;          // above every row and every complement of one
    xent_rows_kernel<<<N, 128, 0, st>>>(target, ignore_index, V, D, target_rest, dloss, reduction == RGB200_REDUCE_NONE, inv_count, W, weight, coefficient,
                                        first, not_last, dX);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;

    EpilogueParams E = {};
    E.target = target; E.lse = lse; E.row_scale = weight;
    EpilogueParams add = {};
    add.residual = dX;
    int* status = reinterpret_cast<int*>(ws + L.status);
    for (int at = 0; at < V; at += L.words) {
        const int words = V - at < L.words ? V - at : L.words;
        const float* Wp = W + (size_t)at * D;
        E.first_word = at;
        E.ldc = both ? padded_words(words) : words;
        if (both) {
            E.row_max = reinterpret_cast<unsigned*>(ws + L.maxima);
            E.col_max = E.row_max + N;
            if (at > 0 && (e = cudaMemsetAsync(E.row_max, 0, maxima_bytes, st)) != cudaSuccess) return e;
        }
        if ((e = gemm_with_epilogue(X, Wp, P, N, words, D, product_config(slices, false, true), EPI_PROB, E,
                                    Prepared{at > 0 && words == L.words, false, status}, ws + L.logits, L.logits_bytes, st)) != cudaSuccess)
            return e;
        const rgb200_config cx = product_config(slices, false, false);
        if (both) {                                  // P once for both products
            PlaneSlots rows, cols;
            if ((e = plane_slots(N, D, words, cx, ws + L.dx, &rows)) != cudaSuccess || (e = plane_slots(words, D, N, product_config(slices, true, false), ws + L.dw, &cols)) != cudaSuccess)
                return e;
            if ((e = launch_split_both(slices, P, E.ldc, N, words, E.row_max, E.col_max, rows, cols, st)) != cudaSuccess) return e;
        }
        // A row that counts and meets a value that is not finite has a P of NaN; X and W need no marks of their own, and must not have them: the rows
        // that do not count take no part, whatever they hold
        if (dX && (e = gemm_with_epilogue(P, Wp, dX, N, D, words, cx, EPI_LINEAR, add, Prepared{both, false, status, false, NF_MARK, NF_UNDEFINED}, ws + L.dx,
                                          L.dx_bytes, st)) != cudaSuccess)
            return e;
        if (dW && (e = transposed_product(P, X, dW + (size_t)at * D, words, D, N, slices, Prepared{both, at > 0 && !transposed_in_ranges(N, slices), status, false, NF_MARK, NF_DROP},
                                          ws + L.dw, L.dw_bytes, st)) != cudaSuccess)
            return e;
    }
    if (dW) {
        xent_single_dw_kernel<<<(N + 7) / 8, 256, 0, st>>>(target, coefficient, X, first, not_last, N, V, D, dW, list, listed);
        // at most N / 2 words are listed; the CTAs walk over them
        const long long most = ((long long)N / 2) * ((D + XENT_DW_COLS - 1) / XENT_DW_COLS);
        if (most > 0) xent_repeated_dw_kernel<<<(int)(most < 148 * 8 ? most : 148 * 8), 256, 0, st>>>(target, coefficient, X, not_last, D, dW, list, listed);
    }
    return cudaGetLastError();
}
