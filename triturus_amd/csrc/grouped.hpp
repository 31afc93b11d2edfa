// What the products of ragged groups share: finding a workgroup's tile from sizes that live on the
// device, element types, and the loads that stage a tile.
//
// T rows are cut into E consecutive groups of sizes[e] rows; rows behind the last group are the
// "tail".  The host knows T and E only, so it launches the most tiles that any sizes can make,
// T / BM + min(E + 1, T) of them per column panel, and every wavefront finds its own tile by a prefix sum
// over the sizes (E = 64: one load and six lane steps).  Sizes that do not fit (negative, or past T in
// sum) are clamped there, so no sizes make a kernel leave the tensors.
#pragma once

#include "common.hpp"

namespace trt {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx8 __attribute__((ext_vector_type(8)));

struct Sizes {
    const void *p;  // nullptr: one group of all T rows
    int wide;       // int64 values instead of int32
    int64_t E, T;
};

struct GroupTile {
    int64_t group;   // E: the tail
    int64_t row0;    // first row of the tile
    int64_t rows;    // rows of the group from row0 on (> 0)
    int64_t column;  // column panel
    int parts, part; // the tile is cut into this many, and this one is meant (find_tile with CUT)
};

__device__ __forceinline__ int64_t size_at(const Sizes &s, int64_t e) {
    if (e >= s.E) return 0;
    if (!s.p) return s.T;
    const int64_t v = s.wide ? static_cast<const int64_t *>(s.p)[e] : (int64_t)static_cast<const int32_t *>(s.p)[e];
    return v < 0 ? 0 : (v > s.T ? s.T : v);
}

__device__ __forceinline__ int64_t wave_prefix(int64_t v) {  // inclusive
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int64_t u = __shfl_up(v, d, kWave);
        if (lane_id() >= d) v += u;
    }
    return v;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Rows [start, end) of group e + lane, for a chunk of 64 groups from e on; `before` is the sum of the
// sizes before the chunk and moves on.  Index E is the tail.
__device__ __forceinline__ void chunk_rows(const Sizes &s, int64_t e, int64_t &before, int64_t &start, int64_t &end) {
    const int64_t g = e + lane_id();
    const int64_t incl = before + wave_prefix(size_at(s, g));
    end = incl < s.T ? incl : s.T;
    start = __shfl_up(end, 1, kWave);
    if (lane_id() == 0) start = before < s.T ? before : s.T;
    if (g == s.E) end = s.T;
    if (g > s.E) start = end = s.T;
    before = uniform64(__shfl(incl, kWave - 1, kWave));
}

// The tile of workgroup `wg`, or false when there is none for it.  Tiles are numbered group by group, in
// bands of 8 row tiles with the row tile running fastest (neighbours share a panel of the group's matrix),
// and dealt out to the XCDs in runs of the tiles there ARE: numbering the upper bound instead would
// leave the last XCDs idle.  Wave-uniform.  The launch has fewer than 2^31 workgroups, so do the tiles.
//
// CUT: tiles of which a CU holds one at a time run in rounds of kCus, and a last round of a few tiles would take as long as a
// full one.  Up to kCus / 4 tiles of it are cut into quarters, up to kCus / 2 into halves, which then fill one shorter round
// (8 groups of 16384 rows in all, K = N = 4096, 1088 tiles of 256 x 256: 560 us in 5 rounds, 520 with quarters).
constexpr uint32_t kCus = 256;
template <int BM, bool CUT = false>
__device__ __forceinline__ bool find_tile(const Sizes &s, uint32_t wg, uint32_t columns, GroupTile &t) {
    const int64_t chunks = s.E / kWave + 1;
    int64_t before = 0, start = 0, end = 0;
    uint32_t total = 0;
    for (int64_t c = 0; c < chunks; ++c) {
        chunk_rows(s, c * kWave, before, start, end);
        uint32_t n = (uint32_t)ceil_div(end - start, BM);
#pragma unroll
        for (int d = kWave / 2; d; d /= 2) n += __shfl_xor(n, d, kWave);
        total += n;
    }
    total = __builtin_amdgcn_readfirstlane(total) * columns;
    const uint32_t rest = total % kCus;
    t.parts = !CUT || rest > kCus / 2 ? 1 : rest > kCus / 4 ? 2 : 4;
    t.part = 0;
    const uint32_t whole = t.parts > 1 ? total - rest : total, per_xcd = (whole + kXcds - 1) / kXcds;
    uint32_t id;
    if (wg < per_xcd * kXcds) {
        id = (wg % kXcds) * per_xcd + wg / kXcds;
        if (id >= whole) return false;
        t.parts = 1;
    } else {
        if (t.parts == 1) return false;
        const uint32_t in = wg - whole;  // the parts of a tile on one XCD
        id = whole + in / kXcds / t.parts * kXcds + in % kXcds;
        t.part = in / kXcds % t.parts;
        if (id >= total) return false;
    }
    uint32_t first = 0;  // row tiles before the chunk
    before = 0;
    for (int64_t c = 0; c < chunks; ++c) {
        if (chunks > 1) chunk_rows(s, c * kWave, before, start, end);
        const uint32_t n = (uint32_t)ceil_div(end - start, BM);
        const uint32_t incl = (uint32_t)wave_prefix(n);
        const uint64_t past = __ballot((first + incl) * columns > id);
        if (past) {
            const int who = __builtin_ctzll(past);
            const uint32_t tiles = __builtin_amdgcn_readfirstlane(__shfl(n, who, kWave));
            const uint32_t at = id - (first + __builtin_amdgcn_readfirstlane(__shfl(incl, who, kWave)) - tiles) * columns;
            constexpr uint32_t kBand = 8;
            const uint32_t band = at / (kBand * columns);
            const uint32_t high = tiles - band * kBand < kBand ? tiles - band * kBand : kBand;
            const uint32_t in = at - band * kBand * columns;
            t.group = c * kWave + who;
            t.row0 = uniform64(__shfl(start, who, kWave)) + (int64_t)(band * kBand + in % high) * BM;
            t.rows = uniform64(__shfl(end, who, kWave)) - t.row0;
            t.column = in / high;
            return true;
        }
        first += __builtin_amdgcn_readfirstlane(__shfl(incl, kWave - 1, kWave));
    }
    return false;
}

// Rows [row0, row0 + rows) of one group.
__device__ __forceinline__ void group_rows(const Sizes &s, int64_t e, int64_t &row0, int64_t &rows) {
    int64_t before = 0, start = 0, end = 0;
    for (int64_t c = 0; c <= e / kWave; ++c) chunk_rows(s, c * kWave, before, start, end);
    row0 = uniform64(__shfl(start, (int)(e % kWave), kWave));
    rows = uniform64(__shfl(end, (int)(e % kWave), kWave)) - row0;
}

// Workgroups that find_tile with CUT wants beyond the tiles.
constexpr int64_t kMostCut = 3 * (kCus / 4) + 4 * kXcds;

inline int64_t most_row_tiles(int64_t T, int64_t E, int BM) { return T / BM + (E + 1 < T ? E + 1 : T); }

// ---- 16 bytes of a row -----------------------------------------------------------------------------
// `left` elements of the row remain from p on (<= 0: none).  A full chunk is one load, whatever the
// alignment (global memory takes 16-byte loads from any address); an end of a row that is not a whole
// chunk is read element by element, so nothing behind the row is touched.
template <typename T>
__device__ __forceinline__ uintx4 load_chunk(const T *p, int64_t left) {
    constexpr int V = 16 / sizeof(T);
    uintx4 v = {0, 0, 0, 0};
    if (left >= V) {
        __builtin_memcpy(&v, p, 16);
    } else if (left > 0) {
        T e[V];
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = T(0);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) e[i] = p[i];
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

}  // namespace trt
