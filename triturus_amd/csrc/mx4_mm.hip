// Products of microscaled 4-bit operands on the scaled matrix pipe: c = a b^T over the values that codes and scales
// stand for, one matrix for all rows or one per group of rows (sizes on the device).
//
// Both operands lie along the contraction, so a 128-byte step of a tile's row is 8 blocks of 32 values, and a lane's 16
// bytes of a fragment are one block: v_mfma_scale_f32_32x32x64_f8f6f4 takes them with the block's scale byte and
// multiplies and scales in one instruction at 4 times the rate of 16-bit operands.  Tiles, staging and LDS
// layout are those of gmm.hpp (the INNER layout in bytes); the 8 scale bytes of a row's step go with them as
// one 8-byte word, from which a lane reads the two pairs of its half: blocks 2 kk + (lane >= 32), kk = 0..3.
#include "few.hpp"
#include "mx4.hpp"

namespace trt {

struct Mx4Args {
    const uint8_t *a, *sa, *b, *sb;  // codes and scales; a: values where the kernel quantises them itself
    void *out;
    Sizes sizes;
    int64_t N, K, bytes;        // columns, contraction; bytes of codes in a row (16 per block)
    int64_t lda, ldsa, ldb, ldsb, b_group, sb_group;  // strides in bytes
    uint32_t columns;
    int dtype;  // of c
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

__device__ __forceinline__ uint32_t load_scales4(const uint8_t *p, int64_t left) {
    uint32_t v = 0;
    if (left >= 4) {
        __builtin_memcpy(&v, p, 4);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) v |= (uint32_t)p[i] << (8 * i);
    }
    return v;
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

// Few rows per group (few.hpp): 16 RT rows x 64 columns, the contraction cut over 8 wavefronts.  A wavefront's unit is
// 64 bytes of codes (4 blocks) by 64 columns: lane (n, g) takes block g of columns n, n + 16, .. and a column's 4 scale
// bytes as one word.  A: the type of a's values, which the lane quantises itself on the way (32 neighbours of a
// row: no other lane is needed, and a call is one launch), or uint8_t for codes.
template <typename A, int RT, bool ALIGNED>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_few_kernel(Mx4Args g) {
    __shared__ float lds[FewLds<RT>::FLOATS];
    GroupTile t;
    if (!find_tile<16 * RT>(g.sizes, blockIdx.x, g.columns, t)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id(), m = l & 15, gk = l >> 4;
    const int64_t col0 = t.column * kFewCols, rows = t.rows, cols = g.N - col0;
    const int64_t e = t.group < g.sizes.E ? t.group : 0;
    const int64_t bytes = t.group < g.sizes.E ? g.bytes : 0;  // behind the last group: zeros
    const A *x = reinterpret_cast<const A *>(g.a) + t.row0 * g.lda;
    const uint8_t *sx = g.sa + t.row0 * g.ldsa, *y = g.b + e * g.b_group + col0 * g.ldb, *sy = g.sb + e * g.sb_group + col0 * g.ldsb;

    floatx4 acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    constexpr bool VALUES = sizeof(A) != 1;
    struct Unit {
        A x[RT][VALUES ? 32 : 16];
        uint32_t sx[RT];
        uintx4 y[4];
        uint32_t sy[4];
    };
    auto load = [&](int64_t u, Unit &n) {
        const int64_t left = bytes - u * 64 - gk * 16, blocks = bytes / 16 - u * 4;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = 16 * i + m;
            const bool there = r < rows;
            if constexpr (VALUES) {
                const int64_t k = u * 128 + gk * 32;
                load_values(x + r * g.lda + k, there && left > 0 ? g.K - k : 0, n.x[i]);
            } else {
                load_values(x + r * g.lda + u * 64 + gk * 16, there ? left : 0, n.x[i]);
                n.sx[i] = load_scales4(sx + r * g.ldsa + u * 4, there ? blocks : 0);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = 16 * j + m;
            if constexpr (ALIGNED) {
                const __amdgpu_buffer_rsrc_t r = make_rsrc(y + u * 64, 0x7fffffff);
                n.y[j] = __builtin_amdgcn_raw_buffer_load_b128(r, left > 0 && c < cols ? c * (uint32_t)g.ldb + gk * 16 : 0x80000000u, 0, 0);
            } else {
                n.y[j] = load_chunk(y + c * g.ldb + u * 64 + gk * 16, c < cols ? left : 0);
            }
            n.sy[j] = load_scales4(sy + c * g.ldsb + u * 4, c < cols ? blocks : 0);
        }
    };
    auto multiply = [&](const Unit &n) {
        typedef int intx8 __attribute__((ext_vector_type(8)));
        auto wide = [](uintx4 v) { return intx8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            uintx4 xf;
            uint32_t s;
            if constexpr (VALUES) {
                s = block_scale(top_bits(n.x[i]));
                xf = uintx4{codes_of(n.x[i], s), codes_of(n.x[i] + 8, s), codes_of(n.x[i] + 16, s), codes_of(n.x[i] + 24, s)};
            } else {
                s = n.sx[i] >> (8 * gk);
                __builtin_memcpy(&xf, n.x[i], 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(xf), wide(n.y[j]), acc[i][j], 4, 4, 0, (int)s, 0,
                                                                             (int)(n.sy[j] >> (8 * gk)));
        }
    };
    const int64_t units = ceil_div(bytes, 64);
    Unit a, b;
    int64_t u = wave;
    load(u, a);
    for (; u < units; u += 2 * kFewWaves) {
        load(u + kFewWaves, b);
        multiply(a);
        load(u + 2 * kFewWaves, a);
        multiply(b);
    }
    const auto of = [](int j, int c) { return 16 * j + c; };
    const int64_t at = t.row0 * g.N + col0;
    switch (g.dtype) {
        case TRT_F32: store_few<float, RT>(acc, lds, wave, static_cast<float *>(g.out) + at, g.N, rows, cols, of); break;
        case TRT_F16: store_few<_Float16, RT>(acc, lds, wave, static_cast<_Float16 *>(g.out) + at, g.N, rows, cols, of); break;
        default: store_few<__bf16, RT>(acc, lds, wave, static_cast<__bf16 *>(g.out) + at, g.N, rows, cols, of); break;
    }
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
int launch_mx4_tile(Mx4Args g, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, BN);
    const int64_t blocks = ceil_div(most_row_tiles(g.sizes.T, g.sizes.E, BM) * (int64_t)g.columns, kXcds) * kXcds;
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((mx4_mm_kernel<T, BM, BN, WM, WN, ALIGNED>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, g);
    return (int)hipGetLastError();
}

template <typename A, int RT>
int launch_mx4_few(Mx4Args g, bool aligned, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, kFewCols);
    const int64_t blocks = ceil_div(most_row_tiles(g.sizes.T, g.sizes.E, 16 * RT) * (int64_t)g.columns, kXcds) * kXcds;
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    if (aligned) hipLaunchKernelGGL((mx4_few_kernel<A, RT, true>), dim3((unsigned)blocks), dim3(64 * kFewWaves), 0, s, g);
    else hipLaunchKernelGGL((mx4_few_kernel<A, RT, false>), dim3((unsigned)blocks), dim3(64 * kFewWaves), 0, s, g);
    return (int)hipGetLastError();
}

// RT of the few-row kernel for this many rows per group on average, 0: 128 x 128 tiles.  tile forces 1 + RT, or 1 for 0.
inline int few_row_tiles(int64_t T, int64_t E, int tile) {
    if (tile) return tile - 1;
    const int64_t mean = T / E;
    return mean <= 16 ? 1 : mean <= 32 ? 2 : 0;
}

template <typename T>
int launch_mx4(const Mx4Args &g, hipStream_t s) {
    const bool aligned = ((reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.b) | (uint64_t)g.lda | (uint64_t)g.ldb |
                           (uint64_t)g.b_group) & 15) == 0;
    return aligned ? launch_mx4_tile<T, 128, 128, 2, 2, true>(g, s) : launch_mx4_tile<T, 128, 128, 2, 2, false>(g, s);
}

}  // namespace trt

using namespace trt;

extern "C" size_t trt_mx4_mm_workspace_bytes(int64_t T, int64_t E, int64_t K, int a_type, int tile) {
    if (a_type < 0 || T <= 0 || E <= 0 || K <= 0 || few_row_tiles(T, E, tile) == 1) return 0;
    return (size_t)(T * ceil_div(K, 32) * 17);
}

extern "C" int trt_mx4_mm(const void *a, const void *a_scales, const void *b, const void *b_scales, const void *sizes, void *c, int64_t T,
                          int64_t E, int64_t K, int64_t N, const int64_t sa[2], const int64_t sb[4], int a_type, int dtype,
                          int wide_sizes, int tile, void *workspace, size_t workspace_bytes, void *stream) {
    if (!a || (!a_scales && a_type < 0) || !b || !b_scales || !c || !sa || !sb || T <= 0 || E <= 0 || K <= 0 || N <= 0) return TRT_E_INVALID;
    if (!sizes && E != 1) return TRT_E_INVALID;
    if (a_type > TRT_BF16 || a_type == TRT_F64 || tile < 0 || tile > TRT_MX4_TILES) return TRT_E_INVALID;
    if (dtype != TRT_F32 && dtype != TRT_F16 && dtype != TRT_BF16) return TRT_E_INVALID;
    for (int i = 0; i < 2; ++i)
        if (sa[i] < 0) return TRT_E_LAYOUT;
    for (int i = 0; i < 4; ++i)
        if (sb[i] < 0) return TRT_E_LAYOUT;
    // 256 rows of a tile are addressed with 31-bit byte offsets
    constexpr int64_t kMost = (int64_t)1 << 23;
    if (sa[0] >= kMost || sb[1] >= kMost || N >= kMost || K > 2 * kMost) return TRT_E_RANGE;
    const int few = few_row_tiles(T, E, tile);
    const size_t need = trt_mx4_mm_workspace_bytes(T, E, K, a_type, tile);
    if (need && (!workspace || workspace_bytes < need)) return TRT_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return TRT_E_LAYOUT;
    Mx4Args g = {};
    g.a = static_cast<const uint8_t *>(a), g.sa = static_cast<const uint8_t *>(a_scales);
    g.b = static_cast<const uint8_t *>(b), g.sb = static_cast<const uint8_t *>(b_scales);
    g.out = c, g.dtype = dtype;
    g.sizes = {sizes, wide_sizes, E, T};
    g.N = N, g.K = K, g.bytes = ceil_div(K, 32) * 16;
    g.lda = sa[0], g.ldsa = sa[1], g.b_group = sb[0], g.ldb = sb[1], g.sb_group = sb[2], g.ldsb = sb[3];
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (need) {  // codes, then scales
        uint8_t *codes = static_cast<uint8_t *>(workspace), *scales = codes + T * g.bytes;
        const int status = trt_mx4_quantize(a, codes, scales, T, K, sa[0], a_type, stream);
        if (status) return status;
        g.a = codes, g.sa = scales, g.lda = g.bytes, g.ldsa = g.bytes / 16;
        a_type = -1;
    }
    if (few) {
        const bool aligned = ((reinterpret_cast<uintptr_t>(b) | (uint64_t)g.ldb | (uint64_t)g.b_group) & 15) == 0;
        if (few == 2) return launch_mx4_few<uint8_t, 2>(g, aligned, s);
        switch (a_type) {
            case TRT_F32: return launch_mx4_few<float, 1>(g, aligned, s);
            case TRT_F16: return launch_mx4_few<_Float16, 1>(g, aligned, s);
            case TRT_BF16: return launch_mx4_few<__bf16, 1>(g, aligned, s);
            default: return launch_mx4_few<uint8_t, 1>(g, aligned, s);
        }
    }
    switch (dtype) {
        case TRT_F32: return launch_mx4<float>(g, s);
        case TRT_F16: return launch_mx4<_Float16>(g, s);
        default: return launch_mx4<__bf16>(g, s);
    }
}
