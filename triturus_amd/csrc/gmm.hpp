// Products of ragged groups on the matrix pipe: one workgroup makes a BM x BN tile of the output.
//
//   rows:     c[r, n] = sum_k a[r, k] b[e(r), k, n]     contraction of K terms, the same for every group
//   weights:  d[e, k, n] = sum_{r in e} a[r, k] g[r, n] contraction over the group's own rows
//
// Both walk the contraction in steps of 128 bytes per row of a tile (64 values of 16 bits, 32 of fp32).
// X is the operand that makes the rows of the tile, Y the one that makes its columns; each comes in one of two
// layouts: INNER, where the contracted axis is contiguous (a; b stored N x K), or OUTER, where the output's
// axis is (b stored K x N; both operands of `weights`).  A tile is read from memory 16 bytes a lane into
// registers one step ahead, written to the idle half of a double buffer in LDS during the current step's
// MFMAs, and read from there as MFMA operands:
//   INNER  [row][8 chunks of 16 bytes], chunk c of row r at c ^ (r & 7): the 8 rows that a quarter-wave reads
//          at once lie in 8 different chunks, so all banks work;
//   OUTER  [contracted][row], 16-bit types by the transposing LDS read (ds_read_b64_tr_b16: 4 x 16 values per
//          16 lanes, each lane gets one column), fp32 by 4-byte reads (32 neighbours); rows are 32 bytes
//          longer than their data, so that the 4 rows of a transposing read lie in different banks.
// Sums are fp32; a result is rounded once.  The finished tile goes through LDS, so that rows are
// written 16 bytes a lane.
#pragma once

#include "grouped.hpp"

namespace trt {

enum { kInner = 0, kOuter = 1 };

template <typename T>
struct Mfma;
template <>
struct Mfma<__bf16> {
    static __device__ __forceinline__ floatx16 step(uintx4 x, uintx4 y, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    }
};
template <>
struct Mfma<_Float16> {
    static __device__ __forceinline__ floatx16 step(uintx4 x, uintx4 y, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    }
};
template <>
struct Mfma<float> {
    static __device__ __forceinline__ floatx16 step(uintx4 x, uintx4 y, floatx16 c) {
        const floatx4 u = __builtin_bit_cast(floatx4, x), v = __builtin_bit_cast(floatx4, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(u[i], v[i], c, 0, 0, 0);
        return c;
    }
};

// One operand's share of a step: B rows of the tile, staged by `THREADS` threads.
template <typename T, int LAYOUT, int B, int THREADS>
struct Operand {
    static constexpr int V = 16 / sizeof(T);           // values per chunk
    static constexpr int KT = 128 / sizeof(T);         // contracted values per step
    static constexpr int ROW = LAYOUT == kInner ? 128 : B * (int)sizeof(T) + 32;  // bytes of an LDS row
    static constexpr int LDS = LAYOUT == kInner ? B * 128 : KT * ROW;
    static constexpr int PER_ROW = LAYOUT == kInner ? 8 : B / V;  // chunks per LDS row
    static constexpr int N = B * 8 / THREADS;          // chunks per thread
    static constexpr int ROWS_STEP = THREADS / PER_ROW;
    static_assert(THREADS % PER_ROW == 0 && B * 8 % THREADS == 0, "threads cover whole LDS rows");

    uintx4 reg[N];

    // p: the tile's first value of the step; ld: stride of the strided axis in values; out: rows of the tile that
    // exist; left: contracted values that remain from this step on.
    template <bool ALIGNED>
    __device__ __forceinline__ void load(const T *p, int64_t ld, int64_t out, int64_t left, int tid) {
        const int r = tid / PER_ROW, c = tid % PER_ROW * V;
        const int64_t rows = LAYOUT == kInner ? out : left, in = (LAYOUT == kInner ? left : out) - c;
        if constexpr (ALIGNED) {  // a chunk lies in the row as a whole or not at all; what does not is read as 0
            const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(p, 0x7fffffff);
            const uint32_t row_bytes = (uint32_t)(ld * (int64_t)sizeof(T));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = r + i * ROWS_STEP;
                const uint32_t at = in > 0 && row < rows ? row * row_bytes + (uint32_t)(c * sizeof(T)) : 0x80000000u;
                reg[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = r + i * ROWS_STEP;
                reg[i] = load_chunk(p + row * ld + c, row < rows ? in : 0);
            }
        }
    }

    __device__ __forceinline__ void store(char *lds, int tid) const {
        const int r = tid / PER_ROW, c = tid % PER_ROW;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = r + i * ROWS_STEP;
            const int at = LAYOUT == kInner ? row * ROW + ((c ^ (row & 7)) * 16) : row * ROW + c * 16;
            *reinterpret_cast<uintx4 *>(lds + at) = reg[i];
        }
    }

    // The lane's 16 bytes for sub-step kk (0..3) and the 32 rows from `row` on: contracted chunk 2 kk + (lane >= 32).
    static __device__ __forceinline__ uintx4 fragment(const char *lds, int row, int kk) {
        const int l = lane_id(), half = l >> 5, m = l & 31;
        if constexpr (LAYOUT == kInner) {
            const int rr = row + m;
            return *reinterpret_cast<const uintx4 *>(lds + rr * ROW + (((2 * kk + half) ^ (rr & 7)) * 16));
        } else if constexpr (sizeof(T) == 2) {
            typedef short short4v __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) short4v *lds4;
            const int k = 16 * kk + 8 * half + ((l & 15) >> 2), col = row + (m & 16) + 4 * (l & 3);
            char *at = const_cast<char *>(lds) + k * ROW + col * 2;
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 4 * ROW));
            const uintx2 a = __builtin_bit_cast(uintx2, lo), b = __builtin_bit_cast(uintx2, hi);
            return uintx4{a[0], a[1], b[0], b[1]};
        } else {
            const char *at = lds + (8 * kk + 4 * half) * ROW + (row + m) * 4;
            uintx4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint32_t *>(at + i * ROW);
            return v;
        }
    }
};

// Waits for the wavefront's own LDS accesses, then for the workgroup's wavefronts; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Writes a finished tile: `out` is its first value, rows x cols of it exist, the output's rows are N long and start at
// `base`.  acc[i][j][q] is row 32 i + (lane & 31), column 32 j + 8 (q / 4) + 4 (lane / 32) + q % 4 of the
// wavefront's part (the MFMA's first operand makes its rows, and that is Y here: 4 neighbours of an output row
// in a lane).  The wavefront turns them round in LDS of its own and writes rows, 16 bytes a lane.
template <typename T, int BM, int BN, int WM, int WN>
struct OutTile {
    static constexpr int ROW = BN / WN * (int)sizeof(T) + 16;  // bytes of a row of a wavefront's part in LDS
    static constexpr int LDS = WM * WN * (BM / WM) * ROW;
};

template <typename T, int BM, int BN, int WM, int WN, int RT, int CT>
__device__ __forceinline__ void store_tile(const floatx16 (&acc)[RT][CT], char *lds, int wave, T *out, int64_t N, int64_t rows,
                                           int64_t cols, const void *base) {
    constexpr int OUT_ROW = OutTile<T, BM, BN, WM, WN>::ROW;
    const int wm = wave / WN, wn = wave % WN, l = lane_id();
    char *mine = lds + wave * (BM / WM) * OUT_ROW;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; q += 4) {
                struct alignas(4 * sizeof(T)) { T v[4]; } four;
#pragma unroll
                for (int u = 0; u < 4; ++u) four.v[u] = (T)acc[i][j][q + u];
                const int row = 32 * i + (l & 31), col = 32 * j + 2 * q + 4 * (l >> 5);
                *reinterpret_cast<decltype(four) *>(mine + row * OUT_ROW + col * sizeof(T)) = four;
            }
    // the wavefront reads what it wrote itself: no barrier
    constexpr int V = 16 / sizeof(T), PER = BN / WN / V, STEP = kWave / PER;
    const int64_t wrows = rows - wm * (BM / WM), wcols = cols - wn * (BN / WN);
    T *dst = out + (int64_t)wm * (BM / WM) * N + wn * (BN / WN);
    const bool whole = ((reinterpret_cast<uintptr_t>(base) | (uint64_t)(N * (int64_t)sizeof(T))) & 15) == 0;
    const int c = l % PER * V;
#pragma unroll 4
    for (int r = l / PER; r < BM / WM; r += STEP) {
        if (r >= wrows || c >= wcols) continue;
        const uintx4 v = *reinterpret_cast<const uintx4 *>(mine + r * OUT_ROW + c * sizeof(T));
        T *p = dst + (int64_t)r * N + c;
        if (whole) {
            *reinterpret_cast<uintx4 *>(p) = v;
        } else {
            T e[V];
            __builtin_memcpy(e, &v, 16);
#pragma unroll
            for (int u = 0; u < V; ++u)
                if (c + u < wcols) p[u] = e[u];
        }
    }
}

struct GmmArgs {
    const void *x, *y;
    void *out;
    Sizes sizes;
    int64_t M, N, K;      // rows: (unused), columns, contraction; weights: rows and columns of a matrix, (unused)
    int64_t ldx, ldy, y_group;  // strides in values; y_group: between the matrices (rows)
    uint32_t row_tiles, columns;  // weights: tiles of a matrix
};

template <typename T, int XL, int YL, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(64 * WM *WN) void gmm_kernel(GmmArgs g) {
    constexpr int THREADS = 64 * WM * WN, RT = BM / WM / 32, CT = BN / WN / 32;
    using X = Operand<T, XL, BM, THREADS>;
    using Y = Operand<T, YL, BN, THREADS>;
    constexpr bool WEIGHTS = XL == kOuter;
    constexpr int KT = X::KT, STAGE = X::LDS + Y::LDS;
    constexpr int OUT = OutTile<T, BM, BN, WM, WN>::LDS;
    __shared__ __attribute__((aligned(16))) char lds[2 * STAGE > OUT ? 2 * STAGE : OUT];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const T *x = static_cast<const T *>(g.x), *y = static_cast<const T *>(g.y);
    T *out = static_cast<T *>(g.out);
    int64_t rows, terms;  // of the tile that exist; of the contraction
    int64_t col0;
    if constexpr (WEIGHTS) {
        const uint32_t per = g.row_tiles * g.columns;
        const uint32_t id = (uint32_t)xcd_logical_id(blockIdx.x, gridDim.x);
        const uint32_t e = id / per, in = id % per;
        if (e >= g.sizes.E) return;
        const int64_t m0 = (int64_t)(in % g.row_tiles) * BM;
        col0 = (int64_t)(in / g.row_tiles) * BN;
        int64_t row0;
        group_rows(g.sizes, e, row0, terms);
        x += row0 * g.ldx + m0;
        y += row0 * g.ldy + col0;
        rows = g.M - m0;
        out += (e * g.M + m0) * g.N + col0;
    } else {
        GroupTile t;
        if (!find_tile<BM>(g.sizes, blockIdx.x, g.columns, t)) return;
        col0 = t.column * BN;
        rows = t.rows;
        terms = t.group < g.sizes.E ? g.K : 0;  // behind the last group: zeros
        x += t.row0 * g.ldx;
        y += (t.group < g.sizes.E ? t.group : 0) * g.y_group + col0 * (YL == kInner ? g.ldy : 1);
        out += t.row0 * g.N + col0;
    }
    const int64_t cols = g.N - col0;
    const int64_t x_step = XL == kInner ? KT : KT * g.ldx, y_step = YL == kInner ? KT : KT * g.ldy;

    floatx16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

    const int wm = wave / WN, wn = wave % WN;
    X xs;
    Y ys;
    const int64_t steps = ceil_div(terms, KT);
    if (steps > 0) {
        xs.template load<ALIGNED>(x, g.ldx, rows, terms, tid);
        ys.template load<ALIGNED>(y, g.ldy, cols, terms, tid);
        xs.store(lds, tid);
        ys.store(lds + X::LDS, tid);
        if (steps > 1) {
            xs.template load<ALIGNED>(x + x_step, g.ldx, rows, terms - KT, tid);
            ys.template load<ALIGNED>(y + y_step, g.ldy, cols, terms - KT, tid);
        }
        lds_barrier();
    }
    for (int64_t s = 0; s < steps; ++s) {
        const char *xl = lds + (s & 1) * STAGE, *yl = xl + X::LDS;
        char *next = lds + ((s + 1) & 1) * STAGE;
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
                for (int j = 0; j < CT; ++j) acc[i][j] = Mfma<T>::step(yf[j], xf[i], acc[i][j]);
            if (kk == 0 && s + 1 < steps) {
                xs.store(next, tid);
                ys.store(next + X::LDS, tid);
                if (s + 2 < steps) {
                    const int64_t left = terms - (s + 2) * KT;
                    xs.template load<ALIGNED>(x + (s + 2) * x_step, g.ldx, rows, left, tid);
                    ys.template load<ALIGNED>(y + (s + 2) * y_step, g.ldy, cols, left, tid);
                }
            }
        }
        lds_barrier();
    }

    store_tile<T, BM, BN, WM, WN>(acc, lds, wave, out, g.N, rows, cols, g.out);
}

}  // namespace trt
