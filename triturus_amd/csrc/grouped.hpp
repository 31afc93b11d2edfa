// What the products of ragged groups share: finding a workgroup's tile from sizes that live on the
// device, element types, and the loads that stage a tile.
//
// T rows are cut into E consecutive groups of sizes[e] rows; rows behind the last group are the
// "tail".  The host knows T and E only, so it launches the most tiles that any sizes can make,
// T / BM + min(E + 1, T) of them per column panel, and every wavefront finds its own tile by a prefix sum
// over the sizes (one load and a few vector instructions for 64 groups).  Sizes that do not fit (negative, or past T in
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

// T < 2^31 (checked by the host), so rows are 32-bit numbers; sums of clamped sizes saturate.
__device__ __forceinline__ uint32_t size_at(const Sizes &s, uint32_t e) {
    const uint32_t T = (uint32_t)s.T;
    if (e >= s.E) return 0;
    if (!s.p) return T;
    const int64_t v = s.wide ? static_cast<const int64_t *>(s.p)[e] : (int64_t)static_cast<const int32_t *>(s.p)[e];
    return v < 0 ? 0 : (v > (int64_t)T ? T : (uint32_t)v);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_zero(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0u, v, CTRL, ROWS, 0xf, false);
}
// Inclusive prefix sum over the wavefront, six vector instructions deep (moves within rows of 16, then of whole rows).
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
    v = __builtin_elementwise_add_sat(v, dpp_or_zero<0x111, 0xf>(v));  // row_shr 1, 2, 4, 8
    v = __builtin_elementwise_add_sat(v, dpp_or_zero<0x112, 0xf>(v));
    v = __builtin_elementwise_add_sat(v, dpp_or_zero<0x114, 0xf>(v));
    v = __builtin_elementwise_add_sat(v, dpp_or_zero<0x118, 0xf>(v));
    v = __builtin_elementwise_add_sat(v, dpp_or_zero<0x142, 0xa>(v));  // row_bcast 15: into rows 1 and 3
    v = __builtin_elementwise_add_sat(v, dpp_or_zero<0x143, 0xc>(v));  // row_bcast 31: into rows 2 and 3
    return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Rows [start, end) of group e + lane, for a chunk of 64 groups from e on; `before` is the sum of the
// sizes before the chunk and moves on.  Index E is the tail.
__device__ __forceinline__ void chunk_rows(const Sizes &s, uint32_t e, uint32_t &before, uint32_t &start, uint32_t &end) {
    const uint32_t g = e + lane_id(), T = (uint32_t)s.T;
    const uint32_t incl = __builtin_elementwise_add_sat(before, wave_prefix(size_at(s, g)));
    const uint32_t first = before < T ? before : T;
    end = incl < T ? incl : T;
    start = __builtin_amdgcn_update_dpp(first, end, 0x138, 0xf, 0xf, false);  // wave_shr 1; lane 0 keeps `first`
    if (g == s.E) end = T;
    if (g > s.E) start = end = T;
    before = lane_value(incl, kWave - 1);
}

// The tile of workgroup `wg`, or false when there is none for it.  Tiles are numbered group by group, in
// bands of 8 row tiles with the row tile running fastest (neighbours share a panel of the group's matrix),
// and dealt out to the XCDs in runs of the tiles there ARE: numbering the upper bound instead would
// leave the last XCDs idle.  Wave-uniform.  The launch has fewer than 2^31 workgroups, so do the tiles.
//
// CUT: tiles of which a CU holds one at a time run in rounds of kCus, and a last round of a few tiles would take as long as a
// full one.  Up to kCus / 4 tiles of it are cut into quarters, up to kCus / 2 into halves, which then fill one shorter round
// (8 groups of 16384 rows in all, K = N = 4096, 1088 tiles of 256 x 256: 560 us in 5 rounds, 541 with
// quarters, before later steps).
constexpr uint32_t kCus = 256;
template <int BM, bool CUT = false>
__device__ __forceinline__ bool find_tile(const Sizes &s, uint32_t wg, uint32_t columns, GroupTile &t) {
    const uint32_t chunks = (uint32_t)s.E / kWave + 1;
    uint32_t before = 0, start = 0, end = 0, total = 0, incl = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
        chunk_rows(s, c * kWave, before, start, end);
        incl = wave_prefix((end - start + (BM - 1)) / BM);
        total += lane_value(incl, kWave - 1);
    }
    total *= columns;
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
    for (uint32_t c = 0; c < chunks; ++c) {
        if (chunks > 1) {
            chunk_rows(s, c * kWave, before, start, end);
            incl = wave_prefix((end - start + (BM - 1)) / BM);
        }
        const uint64_t past = __ballot((first + incl) * columns > id);
        if (past) {
            const int who = __builtin_ctzll(past);
            const uint32_t start_row = lane_value(start, who), end_row = lane_value(end, who);
            const uint32_t tiles = (end_row - start_row + (BM - 1)) / BM;
            const uint32_t at = id - (first + lane_value(incl, who) - tiles) * columns;
            constexpr uint32_t kBand = 8;
            const uint32_t band = at / (kBand * columns);
            const uint32_t high = tiles - band * kBand < kBand ? tiles - band * kBand : kBand;
            const uint32_t in = at - band * kBand * columns;
            t.group = c * kWave + who;
            t.row0 = start_row + (band * kBand + in % high) * BM;
            t.rows = end_row - t.row0;
            t.column = in / high;
            return true;
        }
        first += lane_value(incl, kWave - 1);
    }
    return false;
}

// Rows [row0, row0 + rows) of the group that stands at place e by length, the longest first, and its number; up to 64 groups.
__device__ __forceinline__ uint32_t group_by_length(const Sizes &s, uint32_t e, int64_t &row0, int64_t &rows) {
    uint32_t before = 0, start = 0, end = 0, place = 0;
    chunk_rows(s, 0, before, start, end);
    const uint32_t mine = (uint32_t)lane_id() < s.E ? end - start : 0;
    for (uint32_t i = 0; i < s.E; ++i) {
        const uint32_t other = lane_value(mine, i);
        place += other > mine || (other == mine && i < (uint32_t)lane_id());
    }
    const int who = __builtin_ctzll(__ballot(place == e && (uint32_t)lane_id() < s.E));
    row0 = lane_value(start, who);
    rows = lane_value(end, who) - row0;
    return who;
}

// Rows [row0, row0 + rows) of one group.
__device__ __forceinline__ void group_rows(const Sizes &s, uint32_t e, int64_t &row0, int64_t &rows) {
    uint32_t before = 0, start = 0, end = 0;
    for (uint32_t c = 0; c <= e / kWave; ++c) chunk_rows(s, c * kWave, before, start, end);
    row0 = lane_value(start, e % kWave);
    rows = lane_value(end, e % kWave) - row0;
}

// Workgroups that find_tile with CUT wants beyond the tiles.
constexpr int64_t kMostCut = 3 * (kCus / 4) + 4 * kXcds;

inline int64_t most_row_tiles(int64_t T, int64_t E, int BM) { return T / BM + (E + 1 < T ? E + 1 : T); }

// n / d for n < 2^31 by one multiplication (d fixed by the host).
struct Divider {
    uint32_t d, m, s;
};
inline Divider divider(uint32_t d) {
    uint32_t s = 0;
    while (((uint64_t)1 << s) < d) ++s;
    return {d, (uint32_t)(((((uint64_t)1 << s) - d) << 32) / d + 1), s};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider &v) { return (__umulhi(n, v.m) + n) >> v.s; }

// Groups cut into pieces of len.d rows, the last one of a group shorter, numbered through all groups.  The first lane `want(first,
// count)` holds for, over all groups' first pieces and their numbers of pieces, says which group it is; rows [start, end) are its own.
struct GroupPieces {
    uint32_t first, count, start, end;
};
template <typename F>
__device__ __forceinline__ bool find_pieces(const Sizes &s, const Divider &len, GroupPieces &p, F want) {
    uint32_t before = 0, start = 0, end = 0, pieces = 0;
    for (uint32_t e = 0; e < s.E; e += kWave) {
        chunk_rows(s, e, before, start, end);
        const bool there = e + lane_id() < s.E;
        const uint32_t n = there ? end - start : 0, count = n ? divide(n - 1, len) + 1 : 0, incl = wave_prefix(count);
        const uint64_t mask = __ballot(there && want(e + lane_id(), pieces + incl - count, count));
        if (mask) {
            const int who = __builtin_ctzll(mask);
            p = {lane_value(pieces + incl - count, who), lane_value(count, who), lane_value(start, who), lane_value(end, who)};
            return true;
        }
        pieces += lane_value(incl, kWave - 1);
    }
    return false;
}

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
// The same way back: `left` > 0 values of the row from p on.
template <typename T>
__device__ __forceinline__ void store_chunk(T *p, uintx4 v, int64_t left) {
    constexpr int V = 16 / sizeof(T);
    if (left >= V) {
        __builtin_memcpy(p, &v, 16);
    } else {
        T e[V];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int i = 0; i < V - 1; ++i)
            if (i < left) p[i] = e[i];
    }
}

}  // namespace trt
