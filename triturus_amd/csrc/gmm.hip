// C entries of the products of ragged groups (kernels: gmm.hpp, one translation unit per element type).
#include "gmm_launch.hpp"

using namespace trt;

namespace {

// 256 rows of a tile are addressed with 31-bit byte offsets
bool stride_fits(int64_t ld, size_t size) { return ld >= 0 && ld * (int64_t)size * 256 < ((int64_t)1 << 31); }

size_t type_size(int dtype) { return dtype == TRT_F32 ? 4 : (dtype == TRT_F16 || dtype == TRT_BF16) ? 2 : 0; }

int dispatch(const GmmArgs &g, int64_t E, int64_t T, bool weights, bool y_inner, int dtype, int tile, void *stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TRT_BF16: return gmm_bf16(g, E, T, weights, y_inner, tile, s);
        case TRT_F16: return gmm_f16(g, E, T, weights, y_inner, tile, s);
        default: return gmm_f32(g, E, T, weights, y_inner, tile, s);
    }
}

}  // namespace

extern "C" int trt_gmm(const void *a, const void *b, const void *sizes, void *c, int64_t T, int64_t E, int64_t K, int64_t N,
                       int64_t lda, const int64_t sb[3], int dtype, int wide_sizes, int tile, void *stream) {
    const size_t size = type_size(dtype);
    if (!a || !b || !sizes || !c || !sb || T <= 0 || E <= 0 || K <= 0 || N <= 0 || !size || tile < 0 || tile > TRT_GMM_TILES)
        return TRT_E_INVALID;
    if (lda < 0 || sb[0] < 0 || sb[1] < 0 || sb[2] < 0) return TRT_E_LAYOUT;
    const bool inner = sb[1] == 1;
    if (!inner && sb[2] != 1) return TRT_E_LAYOUT;
    const int64_t ldb = inner ? sb[2] : sb[1];
    if (!stride_fits(lda, size) || !stride_fits(ldb, size) || !stride_fits(N, size) || !stride_fits(K, size)) return TRT_E_RANGE;
    GmmArgs g = {};
    g.x = a, g.y = b, g.out = c;
    g.sizes = {sizes, wide_sizes, E, T};
    g.N = N, g.K = K, g.ldx = lda, g.ldy = ldb, g.y_group = sb[0];
    return dispatch(g, E, T, false, inner, dtype, tile, stream);
}

extern "C" int trt_gmm_weights(const void *a, const void *g_, const void *sizes, void *d, int64_t T, int64_t E, int64_t K,
                               int64_t N, int64_t lda, int64_t ldg, int dtype, int wide_sizes, int tile, void *stream) {
    const size_t size = type_size(dtype);
    if (!a || !g_ || !sizes || !d || T <= 0 || E <= 0 || K <= 0 || N <= 0 || !size || tile < 0 || tile > TRT_GMM_TILES)
        return TRT_E_INVALID;
    if (lda < 0 || ldg < 0) return TRT_E_LAYOUT;
    if (!stride_fits(lda, size) || !stride_fits(ldg, size) || !stride_fits(N, size) || !stride_fits(K, size)) return TRT_E_RANGE;
    GmmArgs g = {};
    g.x = a, g.y = g_, g.out = d;
    g.sizes = {sizes, wide_sizes, E, T};
    g.M = K, g.N = N, g.ldx = lda, g.ldy = ldg;
    return dispatch(g, E, T, true, false, dtype, tile, stream);
}
