// Products of microscaled 4-bit operands on the scaled matrix pipe: c = a b^T over the values that codes and scales
// stand for, one matrix for all rows or one per group of rows (sizes on the device).
//
// Both operands lie along the contraction, so a 128-byte step of a tile's row is 8 blocks of 32 values, and a lane's 16
// bytes of a fragment are one block: v_mfma_scale_f32_32x32x64_f8f6f4 takes them with the block's scale byte and
// multiplies and scales in one instruction at 4 times the rate of 16-bit operands.  Tiles, staging and LDS
// layout are those of gmm.hpp (the INNER layout in bytes); the 8 scale bytes of a row's step go with them as
// one 8-byte word, from which a lane reads the two pairs of its half: blocks 2 kk + (lane >= 32), kk = 0..3.
#include "gmm.hpp"

namespace trt {

struct Mx4Args {
    const uint8_t *a, *sa, *b, *sb;  // codes and scales
    void *out;
    Sizes sizes;
    int64_t N, bytes;           // columns; bytes of codes in a row (16 per block)
    int64_t lda, ldsa, ldb, ldsb, b_group, sb_group;  // strides in bytes
    uint32_t columns;
};

__device__ __forceinline__ uintx2 load_scales(const uint8_t *p, int64_t left) {
    uint64_t v = 0;
    if (left >= 8) {
        __builtin_memcpy(&v, p, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) v |= (uint64_t)p[i] << (8 * i);
    }
    return __builtin_bit_cast(uintx2, v);
}

template <int PAIR>
__device__ __forceinline__ floatx16 mx4_mfma(uintx4 x, uint32_t sx, uintx4 y, uint32_t sy, floatx16 c) {
    typedef int intx8 __attribute__((ext_vector_type(8)));
    const intx8 u = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0}, v = {(int)y[0], (int)y[1], (int)y[2], (int)y[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(u, v, c, 4, 4, 2 * PAIR, (int)sx, 2 * PAIR, (int)sy);
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(64 * WM *WN) void mx4_mm_kernel(Mx4Args g) {
    constexpr int THREADS = 64 * WM * WN, RT = BM / WM / 32, CT = BN / WN / 32;
    using X = Operand<uint8_t, kInner, BM, THREADS>;
    using Y = Operand<uint8_t, kInner, BN, THREADS>;
    constexpr int CODES = X::LDS + Y::LDS, STAGE = CODES + (BM + BN) * 8, OUT = OutTile<T, BM, BN, WM, WN>::LDS;
    constexpr int NS = (BM + BN) / THREADS;  // scale words of a thread
    static_assert((BM + BN) % THREADS == 0 && BM % THREADS == 0 || THREADS == BM + BN, "a thread's scales are of one operand");
    __shared__ __attribute__((aligned(16))) char lds[2 * STAGE > OUT ? 2 * STAGE : OUT];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    GroupTile t;
    if (!find_tile<BM>(g.sizes, blockIdx.x, g.columns, t)) return;
    const int64_t col0 = t.column * BN, rows = t.rows, cols = g.N - col0;
    const int64_t e = t.group < g.sizes.E ? t.group : 0;
    const int64_t bytes = t.group < g.sizes.E ? g.bytes : 0;  // behind the last group: zeros
    const uint8_t *x = g.a + t.row0 * g.lda, *y = g.b + e * g.b_group + col0 * g.ldb;
    const uint8_t *sx = g.sa + t.row0 * g.ldsa, *sy = g.sb + e * g.sb_group + col0 * g.ldsb;

    floatx16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

    const int wm = wave / WN, wn = wave % WN, l = lane_id();
    X xs;
    Y ys;
    uintx2 scales[NS];
    auto load = [&](int64_t s) {
        const int64_t left = bytes - s * 128;
        xs.template load<ALIGNED>(x + s * 128, g.lda, rows, left, tid);
        ys.template load<ALIGNED>(y + s * 128, g.ldb, cols, left, tid);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int r = tid + i * THREADS;
            const bool of_x = r < BM;
            const int64_t row = of_x ? r : r - BM;
            const bool there = row < (of_x ? rows : cols);
            const uint8_t *p = (of_x ? sx + row * g.ldsa : sy + row * g.ldsb) + s * 8;
            scales[i] = load_scales(p, there ? left / 16 : 0);
        }
    };
    auto store = [&](char *to) {
        xs.store(to, tid);
        ys.store(to + X::LDS, tid);
#pragma unroll
        for (int i = 0; i < NS; ++i) *reinterpret_cast<uintx2 *>(to + CODES + (tid + i * THREADS) * 8) = scales[i];
    };
    const int64_t steps = ceil_div(bytes, 128);
    if (steps > 0) {
        load(0);
        store(lds);
        if (steps > 1) load(1);
        lds_barrier();
    }
    for (int64_t s = 0; s < steps; ++s) {
        const char *xl = lds + (s & 1) * STAGE, *yl = xl + X::LDS, *sl = xl + CODES;
        char *next = lds + ((s + 1) & 1) * STAGE;
        uintx2 xe[RT], ye[CT];
        const int half = 8 * (l >> 5);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uintx2 v = *reinterpret_cast<const uintx2 *>(sl + ((wm * RT + i) * 32 + (l & 31)) * 8);
            xe[i] = uintx2{v[0] >> half, v[1] >> half};
        }
#pragma unroll
        for (int j = 0; j < CT; ++j) {
            const uintx2 v = *reinterpret_cast<const uintx2 *>(sl + (BM + (wn * CT + j) * 32 + (l & 31)) * 8);
            ye[j] = uintx2{v[0] >> half, v[1] >> half};
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uintx4 xf[RT], yf[CT];
#pragma unroll
            for (int i = 0; i < RT; ++i) xf[i] = X::fragment(xl, (wm * RT + i) * 32, kk);
#pragma unroll
            for (int j = 0; j < CT; ++j) yf[j] = Y::fragment(yl, (wn * CT + j) * 32, kk);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < CT; ++j)
                    acc[i][j] = kk & 1 ? mx4_mfma<1>(yf[j], ye[j][kk / 2], xf[i], xe[i][kk / 2], acc[i][j])
                                       : mx4_mfma<0>(yf[j], ye[j][kk / 2], xf[i], xe[i][kk / 2], acc[i][j]);
            if (kk == 0 && s + 1 < steps) {
                store(next);
                if (s + 2 < steps) load(s + 2);
            }
        }
        lds_barrier();
    }
    T *out = static_cast<T *>(g.out) + t.row0 * g.N + col0;
    store_tile<T, BM, BN, WM, WN>(acc, lds, wave, out, g.N, rows, cols, g.out);
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
int launch_mx4_tile(Mx4Args g, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, BN);
    const int64_t blocks = ceil_div(most_row_tiles(g.sizes.T, g.sizes.E, BM) * (int64_t)g.columns, kXcds) * kXcds;
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((mx4_mm_kernel<T, BM, BN, WM, WN, ALIGNED>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, g);
    return (int)hipGetLastError();
}

template <typename T>
int launch_mx4(const Mx4Args &g, hipStream_t s) {
    const bool aligned = ((reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.b) | (uint64_t)g.lda | (uint64_t)g.ldb |
                           (uint64_t)g.b_group) & 15) == 0;
    return aligned ? launch_mx4_tile<T, 128, 128, 2, 2, true>(g, s) : launch_mx4_tile<T, 128, 128, 2, 2, false>(g, s);
}

}  // namespace trt

using namespace trt;

extern "C" int trt_mx4_mm(const void *a, const void *a_scales, const void *b, const void *b_scales, const void *sizes, void *c, int64_t T,
                          int64_t E, int64_t K, int64_t N, const int64_t sa[2], const int64_t sb[4], int dtype, int wide_sizes,
                          void *stream) {
    if (!a || !a_scales || !b || !b_scales || !c || !sa || !sb || T <= 0 || E <= 0 || K <= 0 || N <= 0) return TRT_E_INVALID;
    if (!sizes && E != 1) return TRT_E_INVALID;
    for (int i = 0; i < 2; ++i)
        if (sa[i] < 0) return TRT_E_LAYOUT;
    for (int i = 0; i < 4; ++i)
        if (sb[i] < 0) return TRT_E_LAYOUT;
    // 256 rows of a tile are addressed with 31-bit byte offsets
    constexpr int64_t kMost = (int64_t)1 << 23;
    if (sa[0] >= kMost || sb[1] >= kMost || N >= kMost || K > 2 * kMost) return TRT_E_RANGE;
    Mx4Args g = {};
    g.a = static_cast<const uint8_t *>(a), g.sa = static_cast<const uint8_t *>(a_scales);
    g.b = static_cast<const uint8_t *>(b), g.sb = static_cast<const uint8_t *>(b_scales);
    g.out = c;
    g.sizes = {sizes, wide_sizes, E, T};
    g.N = N, g.bytes = ceil_div(K, 32) * 16;
    g.lda = sa[0], g.ldsa = sa[1], g.b_group = sb[0], g.ldb = sb[1], g.sb_group = sb[2], g.ldsb = sb[3];
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TRT_F32: return launch_mx4<float>(g, s);
        case TRT_F16: return launch_mx4<_Float16>(g, s);
        case TRT_BF16: return launch_mx4<__bf16>(g, s);
        default: return TRT_E_INVALID;
    }
}
