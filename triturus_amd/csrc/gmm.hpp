// Products of ragged groups on the matrix pipe: one workgroup makes a BM x BN tile of the output.
//
//   rows:     c[r, n] = sum_k a[r, k] b[e(r), k, n]     contraction of K terms, the same for every group
//   weights:  d[e, k, n] = sum_{r in e} a[r, k] g[r, n] contraction over the group's own rows
//
// Both walk the contraction in steps of 64 bytes per row of a tile (32 values of 16 bits, 16 of fp32).
// X is the operand that makes the rows of the tile, Y the one that makes its columns; each comes in one of two
// layouts: INNER, where the contracted axis is contiguous (a; b stored N x K), or OUTER, where the output's
// axis is (b stored K x N; both operands of `weights`).  A tile is read from memory 16 bytes a lane into
// registers ahead of its step, written to the idle one of three stages in LDS during the current step's
// MFMAs, and read from there as MFMA operands:
//   INNER  [row][4 chunks of 16 bytes], chunk c of row r at c ^ (r / 4 % 4): four runs of 4 rows, whose chunks are in four
//          different places, fill all 64 banks;
//   OUTER  [contracted][row], 16-bit types by the transposing LDS read (ds_read_b64_tr_b16: 4 x 16 values per
//          16 lanes, each lane gets one column), with row k's pairs of chunks turned by 2 (k % 4) so that the 4 rows and 2 pairs
//          that are read at a time lie in all banks; fp32 by 4-byte reads (32 neighbours) from rows 32 bytes longer than
//          their data.
// (With r / 2 % 4 and turns by k % 4, half of the reads met in a bank: LDS was busy 52 % of the time on 256 x 256 tiles, 26 % so.)
// Sums are fp32; a result is rounded once.  The finished tile goes through LDS, so that rows are
// written 16 bytes a lane.
//
// Bound: the matrix pipe and, on 256 x 256 tiles, the card's power: 16384 rows in 8 groups, K = N = 4096 of bf16 take 437 to 444 us
// (1240 TFLOP/s; matrices stored N x K 460 to 470; the weights' gradient 438 to 443; uneven groups 471 to 493), with the pipe busy
// 69 % of cycles that the clock has stretched to 1.55 GHz.  128 x 128 tiles reach 797 TFLOP/s there (895), fp32 140 (one group of
// 4096 x 4096 x 4096).
#pragma once

#include <utility>

#include "grouped.hpp"

namespace trt {

enum { kInner = 0, kOuter = 1 };
constexpr int kStepBytes = 64, kStages = 3, kSub = kStepBytes / 32;  // sub-steps: MFMAs of 32 bytes per row

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
    static constexpr int KT = kStepBytes / sizeof(T);  // contracted values per step
    static constexpr int CHUNKS = kStepBytes / 16;
    static constexpr int ROW = LAYOUT == kInner ? kStepBytes : B * (int)sizeof(T) + (sizeof(T) == 4 ? 32 : 0);  // bytes of an LDS row
    static constexpr int LDS = LAYOUT == kInner ? B * kStepBytes : KT * ROW;
    static constexpr int PER_ROW = LAYOUT == kInner ? CHUNKS : B / V;  // chunks per LDS row
    static constexpr int N = B * CHUNKS / THREADS;     // chunks per thread
    static constexpr int ROWS_STEP = THREADS / PER_ROW;
    static_assert(THREADS % PER_ROW == 0 && B * CHUNKS % THREADS == 0, "threads cover whole LDS rows");

    // Chunk c of a row of LDS.
    static __device__ __forceinline__ int place(int row, int c) {
        const int turn = LAYOUT == kInner ? (row >> 2) & 3 : sizeof(T) == 4 ? 0 : B >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
        return row * ROW + ((c ^ turn) * 16);
    }

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
        } else if (left >= KT && (LAYOUT == kInner || out >= B)) {
            // every chunk is whole; a row of the tile that does not exist is read as the last one that does, and never written
            const int last = LAYOUT == kInner && out < B ? (int)out - 1 : (LAYOUT == kInner ? B : KT) - 1;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = r + i * ROWS_STEP;
                __builtin_memcpy(&reg[i], p + (row < last ? row : last) * ld + c, 16);
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
            *reinterpret_cast<uintx4 *>(lds + place(r + i * ROWS_STEP, c)) = reg[i];
        }
    }

    // The lane's 16 bytes for sub-step kk and the 32 rows from `row` on: contracted chunk 2 kk + (lane >= 32).
    static __device__ __forceinline__ uintx4 fragment(const char *lds, int row, int kk) {
        const int l = lane_id(), half = l >> 5, m = l & 31;
        if constexpr (LAYOUT == kInner) {
            return *reinterpret_cast<const uintx4 *>(lds + place(row + m, 2 * kk + half));
        } else if constexpr (sizeof(T) == 2) {
            typedef short short4v __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) short4v *lds4;
            const int k = 16 * kk + 8 * half + ((l & 15) >> 2);
            char *at = const_cast<char *>(lds) + place(k, (row + (m & 16)) / 8) + 8 * (l & 3);  // turns are of whole pairs of chunks
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

// Writes a finished tile: `out` is its first value, rows x cols of it exist, the output's rows are N long.  acc[i][j][q] is row 32 i + (lane & 31), column 32 j + 8 (q / 4) + 4 (lane / 32) + q % 4 of the
// wavefront's part (the MFMA's first operand makes its rows, and that is Y here: 4 neighbours of an output row
// in a lane).  The wavefront turns them round in LDS of its own and writes rows, 16 bytes a lane.
template <typename T, int BM, int BN, int WM, int WN>
struct OutTile {
    static constexpr int ROW = BN / WN * (int)sizeof(T) + 16;  // bytes of a row of a wavefront's part in LDS
    static constexpr int LDS = WM * WN * (BM / WM) * ROW;
};

template <typename T, int BM, int BN, int WM, int WN, int RT, int CT>
__device__ __forceinline__ void store_tile(const floatx16 (&acc)[RT][CT], char *lds, int wave, T *out, int64_t N, int64_t rows,
                                           int64_t cols) {
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
    const int c = l % PER * V;
#pragma unroll 4
    for (int r = l / PER; r < BM / WM; r += STEP) {
        if (r >= wrows || c >= wcols) continue;
        const uintx4 v = *reinterpret_cast<const uintx4 *>(mine + r * OUT_ROW + c * sizeof(T));
        T *p = dst + (int64_t)r * N + c;
        store_chunk(p, v, wcols - c);
    }
}

// Asks the scheduler for the block's instructions in turn: LDS writes, loads, LDS reads, MFMAs, an eighth of each at a time.
template <int WRITES, int LOADS, int READS, int MFMAS, int... Q>
__device__ __forceinline__ void interleave(std::integer_sequence<int, Q...>) {
    auto part = [](auto q) {
        constexpr int i = decltype(q)::value, G = sizeof...(Q);
        constexpr int w = WRITES * (i + 1) / G - WRITES * i / G, l = LOADS * (i + 1) / G - LOADS * i / G;
        constexpr int r = READS * (i + 1) / G - READS * i / G, m = MFMAS * (i + 1) / G - MFMAS * i / G;
        if constexpr (w > 0) __builtin_amdgcn_sched_group_barrier(0x200, w, 0);
        if constexpr (l > 0) __builtin_amdgcn_sched_group_barrier(0x020, l, 0);
        if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
        if constexpr (m > 0) __builtin_amdgcn_sched_group_barrier(0x008, m, 0);
    };
    (part(std::integral_constant<int, Q>()), ...);
}
template <int WRITES, int LOADS, int READS, int MFMAS>
__device__ __forceinline__ void interleave() {
    interleave<WRITES, LOADS, READS, MFMAS>(std::make_integer_sequence<int, 8>());
}

struct GmmArgs {
    const void *x, *y;
    void *out;
    Sizes sizes;
    int64_t M, N, K;      // rows: (unused), columns, contraction; weights: rows and columns of a matrix, (unused)
    int64_t ldx, ldy, y_group;  // strides in values; y_group: between the matrices (rows)
    uint32_t row_tiles, columns;  // weights: tiles of a matrix
    Divider piece;                // weights: rows of a piece, whose sums go to `partial`; d = 0: groups are whole
    float *partial;
};

// A piece's sums in the order of the accumulators: 16 bytes a lane, [wavefront][i][j][q / 4][lane].
template <int RT, int CT>
__device__ __forceinline__ void store_partial(const floatx16 (&acc)[RT][CT], float *to, int wave) {
    floatx4 *p = reinterpret_cast<floatx4 *>(to) + wave * (RT * CT * 4 * kWave) + lane_id();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) p[((i * CT + j) * 4 + q) * kWave] = floatx4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
}

// LDS of a tile: the stages, or the finished tile.
template <typename T, int XL, int YL, int BM, int BN, int WM, int WN>
struct GmmLds {
    static constexpr int THREADS = 64 * WM * WN;
    static constexpr int STAGE = Operand<T, XL, BM, THREADS>::LDS + Operand<T, YL, BN, THREADS>::LDS;
    static constexpr int OUT = OutTile<T, BM, BN, WM, WN>::LDS;
    static constexpr int BYTES = kStages * STAGE > OUT ? kStages * STAGE : OUT;
};

// One tile: x, y and out at its first values, rows x cols of it exist, `terms` contracted values.  partial: not null for a piece's sums.
template <typename T, int XL, int YL, int BM, int BN, int WM, int WN, bool ALIGNED>
__device__ __forceinline__ void gmm_tile(const T *x, int64_t ldx, const T *y, int64_t ldy, T *out, int64_t N, int64_t rows, int64_t cols,
                                         int64_t terms, char *lds, float *partial) {
    constexpr int THREADS = 64 * WM * WN, RT = BM / WM / 32, CT = BN / WN / 32;
    using X = Operand<T, XL, BM, THREADS>;
    using Y = Operand<T, YL, BN, THREADS>;
    constexpr int KT = X::KT, STAGE = X::LDS + Y::LDS;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int64_t x_step = XL == kInner ? KT : KT * ldx, y_step = YL == kInner ? KT : KT * ldy;

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
        auto load = [&](int64_t s) {  // behind the last step nothing remains, and nothing is read
            const int64_t left = terms - s * KT;
            xs.template load<ALIGNED>(x + s * x_step, ldx, rows, left, tid);
            ys.template load<ALIGNED>(y + s * y_step, ldy, cols, left, tid);
        };
        auto store = [&](char *to) {
            xs.store(to, tid);
            ys.store(to + X::LDS, tid);
        };
        uintx4 xf[2][RT], yf[2][CT];
        auto fragments = [&](const char *from, int kk) {
#pragma unroll
            for (int i = 0; i < RT; ++i) xf[kk & 1][i] = X::fragment(from, (wm * RT + i) * 32, kk);
#pragma unroll
            for (int j = 0; j < CT; ++j) yf[kk & 1][j] = Y::fragment(from + X::LDS, (wn * CT + j) * 32, kk);
        };
        load(0);
        store(lds);
        load(1);
        store(lds + STAGE);
        load(2);
        lds_barrier();
        fragments(lds, 0);
        char *now = lds, *next = lds + STAGE, *after = lds + 2 * STAGE;
        for (int64_t s = 0; s < steps; ++s) {
#pragma unroll
            for (int kk = 0; kk < kSub; ++kk) {
                constexpr int MF = sizeof(T) == 4 ? 4 : 1;  // MFMAs of a product of fragments
                constexpr int XR = XL == kInner ? 1 : sizeof(T) == 2 ? 2 : 4, YR = YL == kInner ? 1 : sizeof(T) == 2 ? 2 : 4;
                constexpr int READS = RT * XR + CT * YR, MFMAS = RT * CT * MF;
                if (kk == kSub - 1) {
                    store(after);  // the step that was read last: everyone is past the barrier behind it
                    load(s + 3);
                    fragments(next, 0);
                } else {
                    fragments(now, kk + 1);
                }
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < CT; ++j) acc[i][j] = Mfma<T>::step(yf[kk & 1][j], xf[kk & 1][i], acc[i][j]);
                if constexpr (ALIGNED) {
                    if (kk == kSub - 1) interleave<X::N + Y::N, X::N + Y::N, READS, MFMAS>();
                    else interleave<0, 0, READS, MFMAS>();
                }
            }
            lds_barrier();
            char *const read = now;
            now = next, next = after, after = read;
        }
    }
    if (XL == kOuter && partial) return store_partial(acc, partial, wave);
    store_tile<T, BM, BN, WM, WN>(acc, lds, wave, out, N, rows, cols);
}

// ---- 256 x 256 tiles of aligned 16-bit operands: memory to LDS without registers between ----------------------------
typedef __attribute__((address_space(3))) void *lds_ptr;

// One operand's share of a 64-byte step, written by buffer loads that go to LDS: a wavefront's load fills 1 KiB there, lane by
// lane, so the places are fixed and it is the lanes' sources that are permuted.
//   INNER  [row][4 chunks], chunk c of row r at c ^ (r / 4 % 4);
//   OUTER  [contracted][row], the 32 bytes p of contracted value k at p ^ (2 (k % 4)).
template <typename T, int LAYOUT, int B, int WAVES>
struct Direct {
    static constexpr int KT = kStepBytes / sizeof(T);
    static constexpr int ROW = LAYOUT == kInner ? kStepBytes : B * (int)sizeof(T);
    static constexpr int LDS = B * kStepBytes;
    static constexpr int N = LDS / 1024 / WAVES;  // loads of a wavefront
    static_assert(sizeof(T) == 2 && LDS % (1024 * WAVES) == 0, "whole loads for every wavefront");

    uint32_t at[N];  // the lane's byte offset from the step's first value, or beyond the extent where the operand ends
    int depth[N];    // contracted values before the lane's chunk

    __device__ __forceinline__ Direct(int64_t ld, int64_t out, int wave) {
        const int l = lane_id();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int place = (wave * N + i) * 1024 + l * 16, row = place / ROW, slot = place % ROW / 16;
            if constexpr (LAYOUT == kInner) {
                const int c = slot ^ ((row >> 2) & 3);
                depth[i] = c * 8;
                at[i] = row < out ? row * (uint32_t)(ld * sizeof(T)) + c * 16 : 0x80000000u;
            } else {
                const int c = slot ^ (4 * (row & 3));
                depth[i] = row;
                at[i] = c * 8 < out ? row * (uint32_t)(ld * sizeof(T)) + c * 16 : 0x80000000u;
            }
        }
    }

    // base: where the operand's share of a stage begins.  Addresses are one offset from the stage's array: the compiler tells the
    // arrays apart, and so does not wait for one stage's loads when it reads another, only through short chains of them.
    __device__ __forceinline__ void load(const T *p, int64_t left, char *stage, int base, int wave) const {
        const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(p, 0x7fffffff);
#pragma unroll
        for (int i = 0; i < N; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(stage + (base + (wave * N + i) * 1024)), 16, depth[i] < left ? at[i] : 0x80000000u, 0, 0, 0);
    }

    static __device__ __forceinline__ uintx4 fragment(const char *stage, int base, int row, int kk) {
        const int l = lane_id(), half = l >> 5, m = l & 31;
        if constexpr (LAYOUT == kInner) {
            const int r = row + m;
            return *reinterpret_cast<const uintx4 *>(stage + (base + r * ROW + (((2 * kk + half) ^ ((r >> 2) & 3)) * 16)));
        } else {
            typedef short short4v __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) short4v *lds4;
            const int k = 16 * kk + 8 * half + ((l & 15) >> 2), pair = row / 16 + (m >> 4);
            const int at = base + k * ROW + ((pair ^ (2 * (k & 3))) * 32) + 8 * (l & 3);
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) const_cast<char *>(stage + at));
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) const_cast<char *>(stage + (at + 4 * ROW)));
            const uintx2 a = __builtin_bit_cast(uintx2, lo), b = __builtin_bit_cast(uintx2, hi);
            return uintx4{a[0], a[1], b[0], b[1]};
        }
    }
};

// Waits until the wavefront's own LDS reads are done and at most LEFT of its loads are on their way, then for the workgroup.  (A
// release fence would wait for all loads to LDS.)
template <int LEFT>
__device__ __forceinline__ void direct_barrier() {
    static_assert(LEFT < 16, "the low bits of vmcnt");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | LEFT);  // lgkmcnt 0, expcnt any, vmcnt LEFT
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Writes a finished tile (of 16-bit values), 32 rows of a wavefront at a time through 32 x 32 CT values of LDS; 16-byte chunk c of
// row r at c ^ (r % PER).  acc as for store_tile.
template <typename T, int RT, int CT>
__device__ __forceinline__ void store_direct(const floatx16 (&acc)[RT][CT], char *lds, int wave, int wm, int wn, T *out, int64_t N, int64_t rows,
                                             int64_t cols) {
    constexpr int V = 8, PER = CT * 4, STEP = kWave / PER;
    char *mine = lds + wave * (32 * CT * 32 * (int)sizeof(T));
    const int l = lane_id();
    const int64_t wcols = cols - wn * (CT * 32);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t row0 = (wm * RT + i) * 32;
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; q += 4) {
                struct alignas(8) { T v[4]; } four;
#pragma unroll
                for (int u = 0; u < 4; ++u) four.v[u] = (T)acc[i][j][q + u];
                const int row = l & 31, col = 32 * j + 2 * q + 4 * (l >> 5);
                *reinterpret_cast<decltype(four) *>(mine + row * (PER * 16) + (((col / V) ^ (row % PER)) * 16) + col % V * 2) = four;
            }
        const int c = l % PER;
#pragma unroll
        for (int r = l / PER; r < 32; r += STEP) {
            const uintx4 v = *reinterpret_cast<const uintx4 *>(mine + r * (PER * 16) + ((c ^ (r % PER)) * 16));
            if (row0 + r >= rows || c * V >= wcols) continue;
            T *p = out + (row0 + r) * N + wn * (CT * 32) + c * V;
            store_chunk(p, v, wcols - c * V);
        }
    }
}

template <typename T, int XL, int YL, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void gmm_direct_tile(const T *x, int64_t ldx, const T *y, int64_t ldy, T *out, int64_t N, int64_t rows, int64_t cols,
                                                int64_t terms, char *st0, char *st1, char *st2, char *st3) {
    constexpr int RT = BM / WM / 32, CT = BN / WN / 32;
    using X = Direct<T, XL, BM, WM * WN>;
    using Y = Direct<T, YL, BN, WM * WN>;
    constexpr int KT = X::KT;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wm = wave / WN, wn = wave % WN;
    const int64_t x_step = XL == kInner ? KT : KT * ldx, y_step = YL == kInner ? KT : KT * ldy;
    floatx16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
    const int64_t steps = ceil_div(terms, KT);
    if (steps > 0) {
        const X xs(ldx, rows, wave);
        const Y ys(ldy, cols, wave);
        auto load = [&](int64_t s, char *to) {
            const int64_t left = terms - s * KT;
            xs.load(x + s * x_step, left, to, 0, wave);
            ys.load(y + s * y_step, left, to, X::LDS, wave);
        };
        uintx4 xf[2][RT], yf[2][CT];
        auto fragments = [&](const char *from, int kk) {
#pragma unroll
            for (int i = 0; i < RT; ++i) xf[kk][i] = X::fragment(from, 0, (wm * RT + i) * 32, kk);
#pragma unroll
            for (int j = 0; j < CT; ++j) yf[kk][j] = Y::fragment(from, X::LDS, (wn * CT + j) * 32, kk);
        };
        auto multiply = [&](int kk) {
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < CT; ++j) acc[i][j] = Mfma<T>::step(yf[kk][j], xf[kk][i], acc[i][j]);
        };
        constexpr int XR = XL == kInner ? 1 : 2, YR = YL == kInner ? 1 : 2, READS = RT * XR + CT * YR;
        constexpr int LOADS = X::N + Y::N;
        // The barrier stands where the last reads of `now` are done: the loads of the step after the next three go there at once, and
        // have three steps' time.
        auto step = [&](int64_t s, char *now, const char *next) {
            fragments(now, 1);
            multiply(0);
            interleave<0, 0, READS, RT * CT>();
            direct_barrier<2 * LOADS>();  // the loads of the next step have landed
            load(s + 4, now);
            fragments(next, 0);
            multiply(1);
            interleave<0, LOADS, READS, RT * CT>();
        };
        load(0, st0);
        load(1, st1);
        load(2, st2);
        load(3, st3);
        direct_barrier<3 * LOADS>();
        fragments(st0, 0);
        // One way out of the loop: with one behind each step, the compiler joined them before its head, took the loads of any stage
        // to be on their way there, and waited for all of them every fourth step.  (With that, the barrier at the end of a step and
        // half of the time for the loads, uneven groups of the sizes above took 513 us for 499, and the weights' gradient 454 for 441.)
        int64_t s = 0;
        for (; s + 4 <= steps; s += 4) {
            step(s, st0, st1);
            step(s + 1, st1, st2);
            step(s + 2, st2, st3);
            step(s + 3, st3, st0);
        }
        if (s < steps) {
            step(s, st0, st1);
            if (s + 1 < steps) {
                step(s + 1, st1, st2);
                if (s + 2 < steps) step(s + 2, st2, st3);
            }
        }
        direct_barrier<0>();  // nothing is on its way to LDS any more
    }
    store_direct<T, RT, CT>(acc, st0, wave, wm, wn, out, N, rows, cols);
}

// CUT: 256 x 256 tiles whose last, short round is cut into halves or quarters (find_tile).
template <typename T, int XL, int YL, int BM, int BN, int WM, int WN, bool ALIGNED, bool CUT>
__global__ __launch_bounds__(64 * WM *WN) void gmm_kernel(GmmArgs g) {
    static_assert(!CUT || (BM == 256 && BN == 256 && WM == 2 && WN == 4 && XL == kInner), "the parts below");
    constexpr bool DIRECT = ALIGNED && BM == 256 && sizeof(T) == 2;
    constexpr int STAGE = DIRECT ? 512 * kStepBytes : 16;
    __shared__ __attribute__((aligned(1024))) char st0[STAGE], st1[STAGE], st2[STAGE], st3[STAGE];
    __shared__ __attribute__((aligned(16))) char lds[DIRECT ? 16 : GmmLds<T, XL, YL, BM, BN, WM, WN>::BYTES];
    auto tile = [&](auto bm, auto bn, auto wm, auto wn, const T *x, const T *y, T *out, int64_t rows, int64_t cols, int64_t terms,
                    float *partial = nullptr) {
        constexpr int M = decltype(bm)::value, N = decltype(bn)::value, P = decltype(wm)::value, Q = decltype(wn)::value;
        if constexpr (DIRECT) gmm_direct_tile<T, XL, YL, M, N, P, Q>(x, g.ldx, y, g.ldy, out, g.N, rows, cols, terms, st0, st1, st2, st3);
        else gmm_tile<T, XL, YL, M, N, P, Q, ALIGNED>(x, g.ldx, y, g.ldy, out, g.N, rows, cols, terms, lds, partial);
    };
    constexpr std::integral_constant<int, BM> bm;
    constexpr std::integral_constant<int, BN> bn;
    constexpr std::integral_constant<int, WM> wm;
    constexpr std::integral_constant<int, WN> wn;
    const T *x = static_cast<const T *>(g.x), *y = static_cast<const T *>(g.y);
    T *out = static_cast<T *>(g.out);
    if constexpr (XL == kOuter) {
        // Groups differ in length: each one's tiles are dealt out to all XCDs, in runs of neighbours and in bands of 8 row
        // tiles (a run shares panels of both operands in its XCD's L2).  The first run goes to another XCD from
        // group to group, so that matrices of few tiles fill all XCDs too.  (8 groups of 2048 rows on average, K = N = 4096: 1390 us
        // with a group per XCD, 680 us so.)
        const uint32_t per = g.row_tiles * g.columns, run = (per + kXcds - 1) / kXcds;
        uint32_t e = blockIdx.x / kXcds / run;  // or the piece's number
        const uint32_t in = (blockIdx.x + e) % kXcds * run + blockIdx.x / kXcds % run;
        if (in >= per) return;
        constexpr uint32_t kBand = 8;
        const uint32_t band = in / (kBand * g.columns), in_band = in - band * kBand * g.columns;
        const uint32_t high = g.row_tiles - band * kBand < kBand ? g.row_tiles - band * kBand : kBand;
        const int64_t m0 = (int64_t)(band * kBand + in_band % high) * BM, col0 = (int64_t)(in_band / high) * BN;
        int64_t row0, terms;
        float *partial = nullptr;
        if (BM == 128 && g.piece.d) {
            GroupPieces p;
            if (!find_pieces(g.sizes, g.piece, p, [&](uint32_t, uint32_t first, uint32_t count) { return e < first + count; })) return;
            partial = g.partial + ((int64_t)e * per + m0 / BM * g.columns + col0 / BN) * (BM * BN);
            row0 = p.start + (int64_t)(e - p.first) * g.piece.d;
            terms = p.end - row0 < g.piece.d ? p.end - row0 : g.piece.d;
        } else if (g.sizes.E <= kWave) e = group_by_length(g.sizes, e, row0, terms);  // long ones first: the last round is made of short ones
        else group_rows(g.sizes, e, row0, terms);
        tile(bm, bn, wm, wn, x + row0 * g.ldx + m0, y + row0 * g.ldy + col0, out + (e * g.M + m0) * g.N + col0, g.M - m0, g.N - col0, terms, partial);
    } else {
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
        const bool there = t.group < g.sizes.E;  // else behind the last group: zeros
        const int64_t terms = there ? g.K : 0;
        x += t.row0 * g.ldx;
        y += (there ? t.group : 0) * g.y_group + col0 * (YL == kInner ? g.ldy : 1);
        out += t.row0 * g.N + col0;
        if constexpr (CUT) {
            constexpr std::integral_constant<int, 128> half;
            constexpr std::integral_constant<int, 2> two;
            constexpr std::integral_constant<int, 4> four;
            if (t.parts == 4) return tile(half, half, two, four, x, y, out, t.rows, g.N - col0, terms);
            if (t.parts == 2) return tile(bm, half, four, two, x, y, out, t.rows, g.N - col0, terms);
        }
        tile(bm, bn, wm, wn, x, y, out, t.rows, g.N - col0, terms);
    }
}

// The pieces' sums of 128 x 128 tiles (2 x 2 wavefronts), added in order: a workgroup of one wavefront has 32 rows of a wavefront's 64 x 64.
template <typename T>
__global__ __launch_bounds__(kWave) void gmm_join_kernel(GmmArgs g) {
    constexpr int RT = 2, CT = 2;
    using Out = OutTile<T, 32, 32 * CT, 1, 1>;
    __shared__ __attribute__((aligned(16))) char lds[Out::LDS];
    const uint32_t per = g.row_tiles * g.columns, i = blockIdx.x % RT, wave = blockIdx.x / RT % 4, in = blockIdx.x / (RT * 4) % per, e = blockIdx.x / (RT * 4) / per;
    const int64_t row0 = (int64_t)(in / g.columns) * 128 + wave / 2 * 64 + 32 * i, col0 = (int64_t)(in % g.columns) * 128 + wave % 2 * 64;
    if (row0 >= g.M || col0 >= g.N) return;
    GroupPieces own;
    if (!find_pieces(g.sizes, g.piece, own, [&](uint32_t group, uint32_t, uint32_t) { return group == e; })) return;
    const floatx4 *p = reinterpret_cast<const floatx4 *>(g.partial + ((int64_t)own.first * per + in) * (128 * 128)) + (wave * RT + i) * (CT * 4 * kWave) + lane_id();
    const int64_t stride = per * (int64_t)(128 * 128 / 4);
    floatx4 sum[CT * 4] = {};
    constexpr uint32_t AHEAD = 4;  // pieces whose loads are on their way at once
    for (uint32_t piece = 0; piece < own.count; piece += AHEAD, p += AHEAD * stride) {
        floatx4 v[AHEAD][CT * 4];
#pragma unroll
        for (uint32_t a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int q = 0; q < CT * 4; ++q) v[a][q] = piece + a < own.count ? p[a * stride + q * kWave] : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int q = 0; q < CT * 4; ++q) sum[q] += v[a][q];
    }
    floatx16 acc[1][CT];
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[0][j][q] = sum[4 * j + q / 4][q % 4];
    store_tile<T, 32, 32 * CT, 1, 1>(acc, lds, 0, static_cast<T *>(g.out) + ((int64_t)e * g.M + row0) * g.N + col0, g.N, g.M - row0, g.N - col0);
}

}  // namespace trt
