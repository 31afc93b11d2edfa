// Host-side estimates of how long a product of ragged groups takes on each tile, in microseconds.
//
// The host knows T rows in E groups and not their sizes: tiles are counted as if groups were equal, with half a row tile
// lost per group.  `steps` are 64 bytes of the contraction.  The constants are least-squares fits (logarithm of the time) to every
// tile's time on random shapes of 1 to 8192 rows per group: 100 of bf16, 100 of fp32, 80 of the 4-bit format.  The least estimate's
// tile is 2.9 %, 2.5 % and 1.7 % behind the best one on average (34 %, 34 % and 28 % on the worst shape); on 130 and 70 other shapes of bf16
// and fp32 whose operands come from memory 4.3 % and 2.1 % (83 % and 27 %).
#pragma once

#include <math.h>

#include "common.hpp"

namespace trt {

struct GroupedShape {
    double mean, groups, steps;
    int64_t N;
    GroupedShape(int64_t T, int64_t E, int64_t n, int64_t row_bytes)
        : mean((double)T / (double)E), groups((double)(E < T ? E : T)), steps((double)ceil_div(row_bytes, 64)), N(n) {}
    // The groups' matrices once from HBM, at `rate` TB/s (the fits are of matrices that may lie in a cache).
    double stream(double rate) const { return 3.0 + groups * (double)N * steps * 64e-6 / rate; }
    double tiles(int64_t BM, int64_t BN) const {
        const double high = mean / (double)BM + 0.5;
        return groups * (high > 1.0 ? high : 1.0) * (double)ceil_div(N, BN);
    }
};

// 128 x 128: a step with one, two, three workgroups on a CU; rounds of 768.
struct MidCost {
    double one, two, three, fixed, round;
};
inline double estimate(const GroupedShape &g, const MidCost &c) {
    const double n = g.tiles(128, 128), full = floor(n / 768), rest = n - 768 * full;
    const double us = full * c.three + (rest <= 0 ? 0 : rest <= 256 ? c.one : rest <= 512 ? c.two : c.three);
    return c.fixed + g.steps * us + c.round * (full + ceil(rest / 256) / 3);
}

// 256 x 256: a step with a whole tile on each CU, and with halves or quarters in a short last round (find_tile with CUT).
struct BigCost {
    double whole, half, quarter, fixed, round;
};
inline double estimate(const GroupedShape &g, const BigCost &c) {
    const double n = g.tiles(256, 256), full = floor(n / 256), rest = n - 256 * full;
    const double us = rest <= 0 ? 0 : rest <= 64 ? c.quarter : rest <= 128 ? c.half : full > 0 ? c.whole : 0.75 * c.whole;
    return c.fixed + g.steps * (full * c.whole + us) + c.round * (full + (rest <= 0 ? 0 : rest <= 64 ? 0.4 : rest <= 128 ? 0.7 : 1));
}

// 64 x 64: a step of a workgroup alone, and its share of a CU that holds several.
struct SmallCost {
    double alone, shared, fixed;
};
inline double estimate(const GroupedShape &g, const SmallCost &c) {
    const double each = c.shared * ceil(g.tiles(64, 64) / 256);
    return c.fixed + g.steps * (each > c.alone ? each : c.alone);
}

// Few rows: 16 units of a workgroup's wavefronts one after the other, shared once more than `slots` workgroups are there, or the
// matrices' bytes at `rate` TB/s.
struct FewCost {
    double slots, unit, rate, fixed;
};
inline double estimate(const GroupedShape &g, const FewCost &c, int row_tiles) {
    const double n = g.tiles(16 * row_tiles, 64);
    const double chain = ceil(g.steps / 16) * c.unit * (n > c.slots ? n / c.slots : 1.0), read = n * g.steps * 4096e-6 / c.rate;
    return c.fixed + (chain > read ? chain : read);
}

}  // namespace trt
