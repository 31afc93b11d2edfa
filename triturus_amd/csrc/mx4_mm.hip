// Products of microscaled 4-bit operands on the scaled matrix pipe: c = a b^T over the values that codes and scales
// stand for, one matrix for all rows or one per group of rows (sizes on the device).
//
// Both operands lie along the contraction, so a 64-byte step of a tile's row is 4 blocks of 32 values, and a lane's 16
// bytes of a fragment are one block: v_mfma_scale_f32_32x32x64_f8f6f4 takes them with the block's scale byte and
// multiplies and scales in one instruction at 4 times the rate of 16-bit operands.  Tiles, staging and LDS
// layout are those of gmm.hpp (the INNER layout in bytes); the 4 scale bytes of a row's step go with them as
// one word, from which a lane reads the two of its half: blocks 2 kk + (lane >= 32), kk = 0, 1.  In LDS the words lie [step][row],
// so that 32 rows' reads lie in different banks (16 bytes apart, as they come from memory, a dense product took 169 us for 158).
//
// Bound: latency, and a tile's first loads and last stores, beside which a CU has no other tile: 8192 x 4096 by 8192 x 4096 to bf16
// takes 151 to 158 us (3480 to 3640 TFLOP/s), the matrix pipe busy 46 % of cycles at 1.8 GHz and wavefronts waiting for 32 %; 16384
// rows in 8 groups, K = N = 4096, 154 to 162 us (uneven groups 169 to 191).
#include "few.hpp"
#include "mx4.hpp"
#include "tile_cost.hpp"

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

template <typename T, int BM, int BN, int WM, int WN>
struct Mx4Lds {
    static constexpr int THREADS = 64 * WM * WN;
    static constexpr int CODES = Operand<uint8_t, kInner, BM, THREADS>::LDS + Operand<uint8_t, kInner, BN, THREADS>::LDS;
    static constexpr int SCALES = (BM + BN) * 16;  // of four steps
    static constexpr int OUT = OutTile<T, BM, BN, WM, WN>::LDS;
    static constexpr int BYTES = kStages * CODES + 2 * SCALES > OUT ? kStages * CODES + 2 * SCALES : OUT;
};

// One tile: codes x, y and scales sx, sy at its first row and column, `bytes` of codes in a row.
template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
__device__ __forceinline__ void mx4_tile(const Mx4Args &g, const uint8_t *x, const uint8_t *sx, const uint8_t *y, const uint8_t *sy, T *out,
                                         int64_t rows, int64_t cols, int64_t bytes, char *lds) {
    constexpr int THREADS = 64 * WM * WN, RT = BM / WM / 32, CT = BN / WN / 32;
    using X = Operand<uint8_t, kInner, BM, THREADS>;
    using Y = Operand<uint8_t, kInner, BN, THREADS>;
    using L = Mx4Lds<T, BM, BN, WM, WN>;
    constexpr int NS = (BM + BN + THREADS - 1) / THREADS;  // scale words of a thread
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);

    floatx16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

    const int wm = wave / WN, wn = wave % WN, l = lane_id();
    const int64_t steps = ceil_div(bytes, kStepBytes);
    if (steps > 0) {
        X xs;
        Y ys;
        uintx4 scales[NS];
        const int64_t blocks = bytes / 16;
        const uint8_t *sp[NS];  // a row or column that does not exist has the scales of the last one that does, and is not written
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int r = tid + i * THREADS < BM + BN ? tid + i * THREADS : BM + BN - 1;
            const int64_t row = r < BM ? (r < rows ? r : rows - 1) : (r - BM < cols ? r - BM : cols - 1);
            sp[i] = r < BM ? sx + row * g.ldsa : sy + row * g.ldsb;
        }
        char *const ring = lds + kStages * L::CODES;  // scales of four steps, [step][row], and of the next four
        auto load_scales = [&](int64_t q) {
#pragma unroll
            for (int i = 0; i < NS; ++i) scales[i] = load_chunk(sp[i] + q * 16, blocks - q * 16);
        };
        auto store_scales = [&](int64_t q) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (NS * THREADS == BM + BN || tid + i * THREADS < BM + BN)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        *reinterpret_cast<uint32_t *>(ring + (q & 1) * L::SCALES + (u * (BM + BN) + tid + i * THREADS) * 4) = scales[i][u];
        };
        auto load = [&](int64_t s) {  // behind the last step nothing remains, and nothing is read
            const int64_t left = bytes - s * kStepBytes;
            xs.template load<ALIGNED>(x + s * kStepBytes, g.lda, rows, left, tid);
            ys.template load<ALIGNED>(y + s * kStepBytes, g.ldb, cols, left, tid);
        };
        auto store = [&](char *to) {
            xs.store(to, tid);
            ys.store(to + X::LDS, tid);
        };
        uintx4 xf[2][RT], yf[2][CT];
        uint32_t xe[2][RT], ye[2][CT];  // of this step and the next one, moved to the lane's half
        auto fragments = [&](const char *from, int kk) {
#pragma unroll
            for (int i = 0; i < RT; ++i) xf[kk][i] = X::fragment(from, (wm * RT + i) * 32, kk);
#pragma unroll
            for (int j = 0; j < CT; ++j) yf[kk][j] = Y::fragment(from + X::LDS, (wn * CT + j) * 32, kk);
        };
        auto exponents = [&](int64_t s, int which) {
            const char *e = ring + ((s >> 2) & 1) * L::SCALES + (s & 3) * (BM + BN) * 4;
            const int half = 8 * (l >> 5);
#pragma unroll
            for (int i = 0; i < RT; ++i)
                xe[which][i] = *reinterpret_cast<const uint32_t *>(e + ((wm * RT + i) * 32 + (l & 31)) * 4) >> half;
#pragma unroll
            for (int j = 0; j < CT; ++j)
                ye[which][j] = *reinterpret_cast<const uint32_t *>(e + (BM + (wn * CT + j) * 32 + (l & 31)) * 4) >> half;
        };
        load(0);
        load_scales(0);
        store(lds);
        store_scales(0);
        load(1);
        store(lds + L::CODES);
        load(2);
        lds_barrier();
        fragments(lds, 0);
        exponents(0, 0);
        char *now = lds, *next = lds + L::CODES, *after = lds + 2 * L::CODES;
        static_assert(kSub == 2, "two sub-steps: the scale bytes 0 and 2 of the lane's half");
        for (int64_t s0 = 0; s0 < steps; s0 += 4) {
            load_scales(s0 / 4 + 1);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t s = s0 + u;
                if (s >= steps) break;
                fragments(now, 1);
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < CT; ++j) acc[i][j] = mx4_mfma<0>(yf[0][j], ye[u & 1][j], xf[0][i], xe[u & 1][i], acc[i][j]);
                if constexpr (ALIGNED) interleave<0, 0, RT + CT, RT * CT>();
                store(after);  // the step that was read last: everyone is past the barrier behind it
                if (u == 2) store_scales(s0 / 4 + 1);
                load(s + 3);
                fragments(next, 0);
                exponents(s + 1, ~u & 1);
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < CT; ++j) acc[i][j] = mx4_mfma<1>(yf[1][j], ye[u & 1][j], xf[1][i], xe[u & 1][i], acc[i][j]);
                if constexpr (ALIGNED) interleave<X::N + Y::N, X::N + Y::N, 2 * (RT + CT), RT * CT>();
                lds_barrier();
                char *const read = now;
                now = next, next = after, after = read;
            }
        }
    }
    store_tile<T, BM, BN, WM, WN>(acc, lds, wave, out, g.N, rows, cols);
}

// 256 x 256 tiles (and their parts) of codes at 16-byte boundaries: codes from memory to LDS without registers between
// (Direct in gmm.hpp, on codes four at a time), scales of four steps as one 16-byte load a row.
template <typename T, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void mx4_direct_tile(const Mx4Args &g, const uint8_t *x, const uint8_t *sx, const uint8_t *y, const uint8_t *sy, T *out,
                                                int64_t rows, int64_t cols, int64_t bytes, char *st0, char *st1, char *st2, char *st3,
                                                char *ring) {
    constexpr int RT = BM / WM / 32, CT = BN / WN / 32, SCALES = (BM + BN) * 16;
    static_assert(BM + BN <= 64 * WM * WN, "a thread has one row's scales");
    using X = Direct<uint16_t, kInner, BM, WM * WN>;
    using Y = Direct<uint16_t, kInner, BN, WM * WN>;
    constexpr int LOADS = X::N + Y::N;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), wm = wave / WN, wn = wave % WN, l = lane_id();
    floatx16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
    const int64_t steps = ceil_div(bytes, kStepBytes);
    if (steps > 0) {
        const X xs(g.lda / 2, rows, wave);
        const Y ys(g.ldb / 2, cols, wave);
        auto load = [&](int64_t s, char *to) {
            const int64_t left = (bytes - s * kStepBytes) / 2;
            xs.load(reinterpret_cast<const uint16_t *>(x + s * kStepBytes), left, to, 0, wave);
            ys.load(reinterpret_cast<const uint16_t *>(y + s * kStepBytes), left, to, X::LDS, wave);
        };
        const int64_t blocks = bytes / 16;
        const int r = tid < BM + BN ? tid : BM + BN - 1;
        // a row or column that does not exist has the scales of the last one that does, and is not written
        const int64_t row = r < BM ? (r < rows ? r : rows - 1) : (r - BM < cols ? r - BM : cols - 1);
        const uint8_t *sp = r < BM ? sx + row * g.ldsa : sy + row * g.ldsb;
        uintx4 scales;
        auto load_scales = [&](int64_t q) { scales = load_chunk(sp + q * 16, blocks - q * 16); };
        auto store_scales = [&](int64_t q) {
            if (BM + BN < 64 * WM * WN && tid >= BM + BN) return;
#pragma unroll
            for (int u = 0; u < 4; ++u) *reinterpret_cast<uint32_t *>(ring + ((q & 1) * SCALES + (u * (BM + BN) + tid) * 4)) = scales[u];
        };
        uintx4 xf[2][RT], yf[2][CT];
        uint32_t xe[2][RT], ye[2][CT];  // of this step and the next one, moved to the lane's half
        auto fragments = [&](const char *from, int kk) {
#pragma unroll
            for (int i = 0; i < RT; ++i) xf[kk][i] = X::fragment(from, 0, (wm * RT + i) * 32, kk);
#pragma unroll
            for (int j = 0; j < CT; ++j) yf[kk][j] = Y::fragment(from, X::LDS, (wn * CT + j) * 32, kk);
        };
        auto exponents = [&](int64_t s, int which) {
            const int e = (int)((s >> 2) & 1) * SCALES + (int)(s & 3) * (BM + BN) * 4, half = 8 * (l >> 5);
#pragma unroll
            for (int i = 0; i < RT; ++i)
                xe[which][i] = *reinterpret_cast<const uint32_t *>(ring + (e + ((wm * RT + i) * 32 + (l & 31)) * 4)) >> half;
#pragma unroll
            for (int j = 0; j < CT; ++j)
                ye[which][j] = *reinterpret_cast<const uint32_t *>(ring + (e + (BM + (wn * CT + j) * 32 + (l & 31)) * 4)) >> half;
        };
        static_assert(kSub == 2, "two sub-steps: the scale bytes 0 and 2 of the lane's half");
        // U: the step's place in its four.  The scales of the next four are asked for in the first and stored in the third.
        auto step = [&](auto u, int64_t s, char *now, const char *next) {
            constexpr int U = decltype(u)::value;
            if constexpr (U == 0) load_scales(s / 4 + 1);
            fragments(now, 1);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < CT; ++j) acc[i][j] = mx4_mfma<0>(yf[0][j], ye[U & 1][j], xf[0][i], xe[U & 1][i], acc[i][j]);
            interleave<0, 0, RT + CT, RT * CT>();
            direct_barrier<2 * LOADS>();  // the loads of the next step have landed
            load(s + 4, now);
            if constexpr (U == 2) store_scales(s / 4 + 1);
            fragments(next, 0);
            exponents(s + 1, ~U & 1);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < CT; ++j) acc[i][j] = mx4_mfma<1>(yf[1][j], ye[U & 1][j], xf[1][i], xe[U & 1][i], acc[i][j]);
            interleave<0, LOADS, 2 * (RT + CT), RT * CT>();
        };
        load(0, st0);
        load_scales(0);
        store_scales(0);
        load(1, st1);
        load(2, st2);
        load(3, st3);
        direct_barrier<3 * LOADS>();
        fragments(st0, 0);
        exponents(0, 0);
        constexpr std::integral_constant<int, 0> u0;
        constexpr std::integral_constant<int, 1> u1;
        constexpr std::integral_constant<int, 2> u2;
        constexpr std::integral_constant<int, 3> u3;
        int64_t s = 0;  // one way out of the loop, as in gmm_direct_tile
        for (; s + 4 <= steps; s += 4) {
            step(u0, s, st0, st1);
            step(u1, s + 1, st1, st2);
            step(u2, s + 2, st2, st3);
            step(u3, s + 3, st3, st0);
        }
        if (s < steps) {
            step(u0, s, st0, st1);
            if (s + 1 < steps) {
                step(u1, s + 1, st1, st2);
                if (s + 2 < steps) step(u2, s + 2, st2, st3);
            }
        }
        direct_barrier<0>();  // nothing is on its way to LDS any more
    }
    store_direct<T, RT, CT>(acc, st0, wave, wm, wn, out, g.N, rows, cols);
}

// CUT: 256 x 256 tiles whose last, short round is cut into halves or quarters (find_tile).
// DIRECT: codes at 16-byte boundaries, T of 16 bits.
template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED, bool CUT, bool DIRECT>
__global__ __launch_bounds__(64 * WM *WN) void mx4_mm_kernel(Mx4Args g) {
    static_assert(!CUT || (BM == 256 && BN == 256 && WM == 2 && WN == 4), "the parts below");
    constexpr int STAGE = DIRECT ? 512 * kStepBytes : 16;
    __shared__ __attribute__((aligned(1024))) char st0[STAGE], st1[STAGE], st2[STAGE], st3[STAGE], ring[DIRECT ? 2 * 512 * 16 : 16];
    __shared__ __attribute__((aligned(16))) char lds[DIRECT ? 16 : Mx4Lds<T, BM, BN, WM, WN>::BYTES];
    GroupTile t;
    if (!find_tile<BM, CUT>(g.sizes, blockIdx.x, g.columns, t)) return;
    int64_t col0 = t.column * BN;
    if constexpr (CUT) {
        if (t.parts > 1) {
            col0 += (t.part & 1) * (BN / 2);
            t.row0 += (t.part >> 1) * (BM / 2);
            t.rows -= (t.part >> 1) * (BM / 2);
            if (t.rows <= 0 || col0 >= g.N) return;
        }
    }
    const int64_t e = t.group < g.sizes.E ? t.group : 0;
    const int64_t bytes = t.group < g.sizes.E ? g.bytes : 0;  // behind the last group: zeros
    const uint8_t *x = g.a + t.row0 * g.lda, *y = g.b + e * g.b_group + col0 * g.ldb;
    const uint8_t *sx = g.sa + t.row0 * g.ldsa, *sy = g.sb + e * g.sb_group + col0 * g.ldsb;
    T *out = static_cast<T *>(g.out) + t.row0 * g.N + col0;
    auto tile = [&](auto bm, auto bn, auto wm, auto wn) {
        constexpr int M = decltype(bm)::value, N = decltype(bn)::value, P = decltype(wm)::value, Q = decltype(wn)::value;
        if constexpr (DIRECT) mx4_direct_tile<T, M, N, P, Q>(g, x, sx, y, sy, out, t.rows, g.N - col0, bytes, st0, st1, st2, st3, ring);
        else mx4_tile<T, M, N, P, Q, ALIGNED>(g, x, sx, y, sy, out, t.rows, g.N - col0, bytes, lds);
    };
    if constexpr (CUT) {
        constexpr std::integral_constant<int, 128> half;
        constexpr std::integral_constant<int, 2> two;
        constexpr std::integral_constant<int, 4> four;
        if (t.parts == 4) return tile(half, half, two, four);
        if (t.parts == 2) return tile(std::integral_constant<int, 256>(), half, four, two);
    }
    tile(std::integral_constant<int, BM>(), std::integral_constant<int, BN>(), std::integral_constant<int, WM>(), std::integral_constant<int, WN>());
}

// Few rows per group (few.hpp): 16 RT rows x 64 columns, the contraction cut over 8 wavefronts.  A wavefront's unit is
// 64 bytes of codes (4 blocks) by 64 columns: lane (n, g) takes block g of columns n, n + 16, .. and a column's 4 scale
// bytes as one word.  A: the type of a's values, which the lane quantises itself on the way (32 neighbours of a
// row: no other lane is needed, and a call is one launch), or uint8_t for codes.
// FAST: at least 4 blocks in a row.  One row, 4096 x 8192: 8.2 us (17.8 MB at 2.2 TB/s: one round of workgroups, bound by latency).
template <typename A, int RT, bool FAST, int CW = 4, int W = 8, int D = 2>
__global__ __launch_bounds__(64 * W) void mx4_few_kernel(Mx4Args g) {
    constexpr int COLS = 16 * CW;
    __shared__ float lds[FewLds<RT, CW, W>::FLOATS];
    GroupTile t;
    if (!find_tile<16 * RT>(g.sizes, blockIdx.x, g.columns, t)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id(), m = l & 15, gk = l >> 4;
    const int64_t col0 = t.column * COLS, rows = t.rows, cols = g.N - col0;
    const int64_t e = t.group < g.sizes.E ? t.group : 0;
    const int64_t bytes = t.group < g.sizes.E ? g.bytes : 0;  // behind the last group: zeros
    const A *x = reinterpret_cast<const A *>(g.a) + t.row0 * g.lda;
    const uint8_t *sx = g.sa + t.row0 * g.ldsa, *y = g.b + e * g.b_group + col0 * g.ldb, *sy = g.sb + e * g.sb_group + col0 * g.ldsb;

    floatx4 acc[RT][CW];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    constexpr bool VALUES = sizeof(A) != 1;
    struct Unit {
        A x[RT][VALUES ? 32 : 16];
        uint32_t sx[RT];
        uintx4 y[CW];
        uint32_t sy[CW];
        int64_t u;
    };
    auto load = [&](int64_t u, Unit &n) {
        n.u = u;
        if constexpr (FAST) {
            // No branch: a row or column that does not exist is read as the last one that does (and not written), a block
            // behind the last one as the last, under scales made 0: 36 2^-254 at most, which is 0 in fp32.
            const int64_t word = u * 4 < bytes / 16 - 4 ? u * 4 : bytes / 16 - 4, at = u * 64 + gk * 16;
            const int rlast = rows < 16 * RT ? (int)rows - 1 : 16 * RT - 1, clast = cols < COLS ? (int)cols - 1 : COLS - 1;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int r = 16 * i + m < rlast ? 16 * i + m : rlast;
                if constexpr (VALUES) {
                    const int64_t k = u * 128 + gk * 32;
                    __builtin_memcpy(n.x[i], x + r * g.lda + (k < g.K - 32 ? k : g.K - 32), sizeof(n.x[i]));
                    if (u * 128 < g.K && u * 128 + 128 > g.K)  // the unit where the row ends: its last block may not be whole
                        if (k < g.K && k + 32 > g.K) load_values(x + r * g.lda + k, g.K - k, n.x[i]);
                } else {
                    __builtin_memcpy(n.x[i], reinterpret_cast<const uint8_t *>(x) + r * g.lda + (at < bytes - 16 ? at : bytes - 16), 16);
                    __builtin_memcpy(&n.sx[i], sx + r * g.ldsa + word, 4);
                }
            }
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                const int c = 16 * j + m < clast ? 16 * j + m : clast;
                __builtin_memcpy(&n.y[j], y + c * g.ldb + (at < bytes - 16 ? at : bytes - 16), 16);
                __builtin_memcpy(&n.sy[j], sy + c * g.ldsb + word, 4);
            }
        } else {
            const int64_t left = bytes - u * 64 - gk * 16, blocks = bytes / 16 - u * 4;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int r = 16 * i + m;
                if constexpr (VALUES) {
                    const int64_t k = u * 128 + gk * 32;
                    load_values(x + r * g.lda + k, r < rows ? g.K - k : 0, n.x[i]);
                } else {
                    load_values(x + r * g.lda + u * 64 + gk * 16, r < rows ? left : 0, n.x[i]);
                    n.sx[i] = load_scales4(sx + r * g.ldsa + u * 4, r < rows ? blocks : 0);
                }
            }
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                const int c = 16 * j + m;
                n.y[j] = load_chunk(y + c * g.ldb + u * 64 + gk * 16, c < cols ? left : 0);
                n.sy[j] = load_scales4(sy + c * g.ldsb + u * 4, c < cols ? blocks : 0);
            }
        }
    };
    auto multiply = [&](const Unit &n) {
        typedef int intx8 __attribute__((ext_vector_type(8)));
        auto wide = [](uintx4 v) { return intx8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };
        // words read before their place, where the row has ended, are moved down to it
        const int64_t past = FAST && n.u * 4 > bytes / 16 - 4 ? n.u * 4 - (bytes / 16 - 4) : 0;
        const uint32_t down = (uint32_t)(8 * past) & 31, keep = past < 4 ? ~0u : 0u;
        auto scale = [&](uint32_t word) { return ((word >> down) & keep) >> (8 * gk); };
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            uintx4 xf;
            uint32_t s;
            if constexpr (VALUES) {
                s = block_scale(top_bits(n.x[i]));
                uint32_t word[4];
                codes_of(n.x[i], s, word);
                xf = uintx4{word[0], word[1], word[2], word[3]};
                s = n.u * 64 + gk * 16 < bytes ? s : 0;
            } else {
                s = scale(n.sx[i]);
                __builtin_memcpy(&xf, n.x[i], 16);
            }
#pragma unroll
            for (int j = 0; j < CW; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(xf), wide(n.y[j]), acc[i][j], 4, 4, 0, (int)s, 0, (int)scale(n.sy[j]));
        }
    };
    const int64_t units = ceil_div(bytes, 64);
    int64_t u = D * wave;  // neighbours: together whole 128-byte lines of the codes
    if (u < units) {
        Unit n[D];
#pragma unroll
        for (int d = 0; d < D; ++d) load(u + d, n[d]);
        for (; u + W * D < units; u += W * D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                multiply(n[d]);
                load(u + W * D + d, n[d]);
            }
        }
#pragma unroll
        for (int d = 0; d < D; ++d) multiply(n[d]);
    }
    const auto of = [](int j, int c) { return 16 * j + c; };
    const int64_t at = t.row0 * g.N + col0;
    switch (g.dtype) {
        case TRT_F32: store_few<float, RT, CW, W>(acc, lds, wave, static_cast<float *>(g.out) + at, g.N, rows, cols, of); break;
        case TRT_F16: store_few<_Float16, RT, CW, W>(acc, lds, wave, static_cast<_Float16 *>(g.out) + at, g.N, rows, cols, of); break;
        default: store_few<__bf16, RT, CW, W>(acc, lds, wave, static_cast<__bf16 *>(g.out) + at, g.N, rows, cols, of); break;
    }
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED, bool CUT = false, bool DIRECT = false>
int launch_mx4_tile(Mx4Args g, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, BN);
    const int64_t blocks = ceil_div(most_row_tiles(g.sizes.T, g.sizes.E, BM) * (int64_t)g.columns, kXcds) * kXcds + (CUT ? kMostCut : 0);
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((mx4_mm_kernel<T, BM, BN, WM, WN, ALIGNED, CUT, DIRECT>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, g);
    return (int)hipGetLastError();
}

template <typename A, int RT, bool FAST, int CW = 4, int W = 8, int D = 2>
int launch_mx4_few(Mx4Args g, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, 16 * CW);
    const int64_t blocks = ceil_div(most_row_tiles(g.sizes.T, g.sizes.E, 16 * RT) * (int64_t)g.columns, kXcds) * kXcds;
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((mx4_few_kernel<A, RT, FAST, CW, W, D>), dim3((unsigned)blocks), dim3(64 * W), 0, s, g);
    return (int)hipGetLastError();
}

// 16 rows a tile: more and smaller pieces where there are fewer tiles than CUs.
template <typename A>
int launch_mx4_few_rows(const Mx4Args &g, hipStream_t s) {
    if (g.bytes < 64) return launch_mx4_few<A, 1, false>(g, s);
    const double n = GroupedShape(g.sizes.T, g.sizes.E, g.N, 64).tiles(16, kFewCols);
    if (n <= 64) return launch_mx4_few<A, 1, true, 1, 8, 4>(g, s);
    if (n <= 128) return launch_mx4_few<A, 1, true, 2, 8, 4>(g, s);
    return launch_mx4_few<A, 1, true>(g, s);
}

// The few-row kernel quantises a's values itself where its workgroups are few: each makes the codes of its rows again, which costs
// less than a launch up to about a round of workgroups (2 rows, one matrix of 3392 x 4672: 15.0 us a call, 12.4 from
// codes; 8 groups of 6 rows, 7328 x 416: 32 and 17, and the launch takes 2.3 on the GPU and 3 on the host).
inline bool quantizes_on_the_way(int64_t T, int64_t E, int64_t N, int a_type, int tile) {
    return a_type >= 0 && tile == 2 && GroupedShape(T, E, N, 64).tiles(16, kFewCols) <= 300;
}

// Tiles: 1 = 128 x 128, 2, 3 = 16, 32 rows x 64 columns of the few-row kernel, 4 = 256 x 256 (c of 16-bit types); the least of
// the estimated times (tile_cost.hpp), with a launch more where values are quantised before.
inline int choose_mx4_tile(int64_t T, int64_t E, int64_t K, int64_t N, int a_type, int dtype, int tile) {
    if (tile) return tile;
    constexpr MidCost kMid = {0.410, 0.740, 1.634, 4.7, 7.4};
    constexpr BigCost kBig = {0.897, 0.795, 0.445, 3.3, 7.7};
    constexpr FewCost kFew[2] = {{107, 1.10, 4.5, 6.3}, {127, 2.81, 2.7, 5.5}};
    const double launch = a_type >= 0 ? 5.0 : 0.0;
    const GroupedShape g(T, E, N, ceil_div(K, 32) * 16);
    int best = 1;
    double best_us = estimate(g, kMid) + launch;
    auto consider = [&](int t, double us) {
        if (us < best_us) best = t, best_us = us;
    };
    for (int i = 0; i < 2; ++i) consider(2 + i, estimate(g, kFew[i], 1 << i) + (quantizes_on_the_way(T, E, N, a_type, 2 + i) ? 0.0 : launch));
    if (dtype != TRT_F32) consider(4, estimate(g, kBig) + launch);
    return best;
}

template <typename T>
int launch_mx4(const Mx4Args &g, int tile, hipStream_t s) {
    const bool aligned = ((reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.b) | (uint64_t)g.lda | (uint64_t)g.ldb |
                           (uint64_t)g.b_group) & 15) == 0;
    if constexpr (sizeof(T) == 2) {
        if (tile == 4)
            return aligned ? launch_mx4_tile<T, 256, 256, 2, 4, true, true, true>(g, s)
                           : launch_mx4_tile<T, 256, 256, 2, 4, false, true>(g, s);
    }
    return aligned ? launch_mx4_tile<T, 128, 128, 2, 2, true>(g, s) : launch_mx4_tile<T, 128, 128, 2, 2, false>(g, s);
}

}  // namespace trt

using namespace trt;

extern "C" size_t trt_mx4_mm_workspace_bytes(int64_t T, int64_t E, int64_t K, int64_t N, int a_type, int dtype, int tile) {
    if (a_type < 0 || T <= 0 || E <= 0 || K <= 0 || N <= 0) return 0;
    if (quantizes_on_the_way(T, E, N, a_type, choose_mx4_tile(T, E, K, N, a_type, dtype, tile))) return 0;
    return (size_t)(T * ceil_div(K, 32) * 17);
}

extern "C" int trt_mx4_mm(const void *a, const void *a_scales, const void *b, const void *b_scales, const void *sizes, void *c, int64_t T,
                          int64_t E, int64_t K, int64_t N, const int64_t sa[2], const int64_t sb[4], int a_type, int dtype,
                          int wide_sizes, int tile, void *workspace, size_t workspace_bytes, void *stream) {
    if (!a || (!a_scales && a_type < 0) || !b || !b_scales || !c || !sa || !sb || T <= 0 || E <= 0 || K <= 0 || N <= 0) return TRT_E_INVALID;
    if (!sizes && E != 1) return TRT_E_INVALID;
    if (a_type < -1 || a_type > TRT_BF16 || a_type == TRT_F64 || tile < 0 || tile > TRT_MX4_TILES) return TRT_E_INVALID;
    if (dtype != TRT_F32 && dtype != TRT_F16 && dtype != TRT_BF16) return TRT_E_INVALID;
    for (int i = 0; i < 2; ++i)
        if (sa[i] < 0) return TRT_E_LAYOUT;
    for (int i = 0; i < 4; ++i)
        if (sb[i] < 0) return TRT_E_LAYOUT;
    // 256 rows of a tile of codes are addressed with 31-bit byte offsets
    constexpr int64_t kMost = (int64_t)1 << 23;
    if ((a_type < 0 && sa[0] >= kMost) || sb[1] >= kMost || N >= kMost || K > 2 * kMost || T >= (int64_t)1 << 31 || E >= (int64_t)1 << 31) return TRT_E_RANGE;
    const size_t need = trt_mx4_mm_workspace_bytes(T, E, K, N, a_type, dtype, tile);
    tile = choose_mx4_tile(T, E, K, N, a_type, dtype, tile);
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
    if (tile == 2 || tile == 3) {
        if (tile == 3) return g.bytes >= 64 ? launch_mx4_few<uint8_t, 2, true>(g, s) : launch_mx4_few<uint8_t, 2, false>(g, s);
        switch (a_type) {
            case TRT_F32: return launch_mx4_few_rows<float>(g, s);
            case TRT_F16: return launch_mx4_few_rows<_Float16>(g, s);
            case TRT_BF16: return launch_mx4_few_rows<__bf16>(g, s);
            default: return launch_mx4_few_rows<uint8_t>(g, s);
        }
    }
    switch (dtype) {
        case TRT_F32: return launch_mx4<float>(g, tile, s);
        case TRT_F16: return launch_mx4<_Float16>(g, tile, s);
        default: return launch_mx4<__bf16>(g, tile, s);
    }
}
