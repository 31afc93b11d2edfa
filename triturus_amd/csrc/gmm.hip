// C entries of the products of ragged groups (kernels: gmm.hpp, one translation unit per element type).
#include "gmm_launch.hpp"

using namespace trt;

namespace {

// 256 rows of a tile are addressed with 31-bit byte offsets
bool stride_fits(int64_t ld, size_t size) { return ld >= 0 && ld * (int64_t)size * 256 < ((int64_t)1 << 31); }

size_t type_size(int dtype) { return dtype == TRT_F32 ? 4 : (dtype == TRT_F16 || dtype == TRT_BF16) ? 2 : 0; }

int dispatch(const GmmArgs &g, int64_t E, int64_t T, bool weights, bool y_inner, int dtype, int tile, const Workspace &w, void *stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TRT_BF16: return gmm_bf16(g, E, T, weights, y_inner, tile, w, s);
        case TRT_F16: return gmm_f16(g, E, T, weights, y_inner, tile, w, s);
        default: return gmm_f32(g, E, T, weights, y_inner, tile, w, s);
    }
}

// `query`: only the workspace is asked for, without sizes and result.
int rows_args(const void *a, const void *b, const void *sizes, void *c, int64_t T, int64_t E, int64_t K, int64_t N, int64_t lda,
              const int64_t sb[3], int dtype, int wide_sizes, int tile, const void *workspace, bool query, GmmArgs &g, bool &inner) {
    const size_t size = type_size(dtype);
    if (!a || !b || !sb || T <= 0 || E <= 0 || K <= 0 || N <= 0 || !size || tile < 0 || tile > TRT_GMM_TILES) return TRT_E_INVALID;
    if (!query && (!sizes || !c)) return TRT_E_INVALID;
    if (lda < 0 || sb[0] < 0 || sb[1] < 0 || sb[2] < 0 || (reinterpret_cast<uintptr_t>(workspace) & 15)) return TRT_E_LAYOUT;
    inner = sb[1] == 1;
    if (!inner && sb[2] != 1) return TRT_E_LAYOUT;
    const int64_t ldb = inner ? sb[2] : sb[1];
    if (!stride_fits(lda, size) || !stride_fits(ldb, size) || !stride_fits(N, size) || !stride_fits(K, size) || T >= (int64_t)1 << 31 ||
        E >= (int64_t)1 << 31)
        return TRT_E_RANGE;
    g = {};
    g.x = a, g.y = b, g.out = c;
    g.sizes = {sizes, wide_sizes, E, T};
    g.N = N, g.K = K, g.ldx = lda, g.ldy = ldb, g.y_group = sb[0];
    return TRT_OK;
}

int weights_args(const void *a, const void *g_, const void *sizes, void *d, int64_t T, int64_t E, int64_t K, int64_t N, int64_t lda,
                 int64_t ldg, int dtype, int wide_sizes, int tile, const void *workspace, bool query, GmmArgs &g) {
    const size_t size = type_size(dtype);
    if (!a || !g_ || T <= 0 || E <= 0 || K <= 0 || N <= 0 || !size || tile < 0 || tile > TRT_GMM_TILES) return TRT_E_INVALID;
    if (!query && (!sizes || !d)) return TRT_E_INVALID;
    if (lda < 0 || ldg < 0 || (reinterpret_cast<uintptr_t>(workspace) & 15)) return TRT_E_LAYOUT;
    if (!stride_fits(lda, size) || !stride_fits(ldg, size) || !stride_fits(N, size) || !stride_fits(K, size) || T >= (int64_t)1 << 31 ||
        E >= (int64_t)1 << 31)
        return TRT_E_RANGE;
    g = {};
    g.x = a, g.y = g_, g.out = d;
    g.sizes = {sizes, wide_sizes, E, T};
    g.M = K, g.N = N, g.ldx = lda, g.ldy = ldg;
    return TRT_OK;
}

int rows_product(const void *a, const void *b, const void *sizes, void *c, int64_t T, int64_t E, int64_t K, int64_t N, int64_t lda,
                 const int64_t sb[3], int dtype, int wide_sizes, int tile, const Workspace &w, void *stream) {
    GmmArgs g;
    bool inner;
    const int status = rows_args(a, b, sizes, c, T, E, K, N, lda, sb, dtype, wide_sizes, tile, w.p, w.query != nullptr, g, inner);
    return status ? status : dispatch(g, E, T, false, inner, dtype, tile, w, stream);
}

int weights_product(const void *a, const void *g_, const void *sizes, void *d, int64_t T, int64_t E, int64_t K, int64_t N, int64_t lda,
                    int64_t ldg, int dtype, int wide_sizes, int tile, const Workspace &w, void *stream) {
    GmmArgs g;
    const int status = weights_args(a, g_, sizes, d, T, E, K, N, lda, ldg, dtype, wide_sizes, tile, w.p, w.query != nullptr, g);
    return status ? status : dispatch(g, E, T, true, false, dtype, tile, w, stream);
}

// The rows' product with b's last two axes exchanged and the weights' product; the arguments of both are looked at before anything is
// enqueued.
int both_products(const void *g, const void *a, const void *b, const void *sizes, void *da, void *db, int64_t T, int64_t E, int64_t K,
                  int64_t N, int64_t ldg, int64_t lda, const int64_t sb[3], int dtype, int wide_sizes, const Workspace &ws, void *stream) {
    if (!sb) return TRT_E_INVALID;
    const int64_t st[3] = {sb[0], sb[2], sb[1]};
    GmmArgs r, w;
    bool inner;
    const bool query = ws.query != nullptr;
    int status = weights_args(a, g, sizes, db, T, E, K, N, lda, ldg, dtype, wide_sizes, 0, ws.p, query, w);
    if (!status) status = rows_args(g, b, sizes, da, T, E, N, K, ldg, st, dtype, wide_sizes, 0, ws.p, query, r, inner);
    if (status) return status;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TRT_BF16: return gmm_grad_bf16(r, w, E, T, inner, ws, s);
        case TRT_F16: return gmm_grad_f16(r, w, E, T, inner, ws, s);
        default: return gmm_grad_f32(r, w, E, T, inner, ws, s);
    }
}

}  // namespace

extern "C" int trt_gmm(const void *a, const void *b, const void *sizes, void *c, int64_t T, int64_t E, int64_t K, int64_t N,
                       int64_t lda, const int64_t sb[3], int dtype, int wide_sizes, int tile, void *workspace, size_t workspace_bytes,
                       void *stream) {
    return rows_product(a, b, sizes, c, T, E, K, N, lda, sb, dtype, wide_sizes, tile, {workspace, workspace_bytes, nullptr}, stream);
}

extern "C" size_t trt_gmm_workspace_bytes(const void *a, const void *b, int64_t T, int64_t E, int64_t K, int64_t N, int64_t lda,
                                          const int64_t sb[3], int dtype, int tile) {
    size_t bytes = 0;
    rows_product(a, b, nullptr, nullptr, T, E, K, N, lda, sb, dtype, 0, tile, {nullptr, 0, &bytes}, nullptr);
    return bytes;
}

extern "C" int trt_gmm_weights(const void *a, const void *g, const void *sizes, void *d, int64_t T, int64_t E, int64_t K, int64_t N,
                               int64_t lda, int64_t ldg, int dtype, int wide_sizes, int tile, void *workspace, size_t workspace_bytes,
                               void *stream) {
    return weights_product(a, g, sizes, d, T, E, K, N, lda, ldg, dtype, wide_sizes, tile, {workspace, workspace_bytes, nullptr}, stream);
}

extern "C" size_t trt_gmm_weights_workspace_bytes(const void *a, const void *g, int64_t T, int64_t E, int64_t K, int64_t N, int64_t lda,
                                                  int64_t ldg, int dtype, int tile) {
    size_t bytes = 0;
    weights_product(a, g, nullptr, nullptr, T, E, K, N, lda, ldg, dtype, 0, tile, {nullptr, 0, &bytes}, nullptr);
    return bytes;
}

extern "C" int trt_gmm_grad(const void *g, const void *a, const void *b, const void *sizes, void *da, void *db, int64_t T, int64_t E,
                            int64_t K, int64_t N, int64_t ldg, int64_t lda, const int64_t sb[3], int dtype, int wide_sizes, void *workspace,
                            size_t workspace_bytes, void *stream) {
    return both_products(g, a, b, sizes, da, db, T, E, K, N, ldg, lda, sb, dtype, wide_sizes, {workspace, workspace_bytes, nullptr}, stream);
}

extern "C" size_t trt_gmm_grad_workspace_bytes(const void *g, const void *a, const void *b, int64_t T, int64_t E, int64_t K, int64_t N,
                                               int64_t ldg, int64_t lda, const int64_t sb[3], int dtype) {
    size_t bytes = 0;
    both_products(g, a, b, nullptr, nullptr, nullptr, T, E, K, N, ldg, lda, sb, dtype, 0, {nullptr, 0, &bytes}, nullptr);
    return bytes;
}
