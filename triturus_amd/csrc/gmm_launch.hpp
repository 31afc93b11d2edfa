// The choice of a tile for a product of ragged groups, shared by the element types.
#pragma once

#include <math.h>

#include <initializer_list>

#include "few.hpp"

namespace trt {

// Tiles of the rows' products: 1 = 128 x 128, 2, 3, 4 = 16, 32, 64 rows x 64 columns of the few-row kernel, 5 = 256 x 256
// (16-bit types).  Of the weights' gradient: 1 = 128 x 128, 2 = 64 x 64, 5 = 256 x 256.
template <typename T, int XL, int YL, int BM, int BN, int WM, int WN, bool ALIGNED, bool CUT = false>
int launch_gmm_tile(GmmArgs g, int64_t E, int64_t T_rows, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, BN);
    int64_t blocks;
    if (XL == kOuter) {
        g.row_tiles = (uint32_t)ceil_div(g.M, BM);
        blocks = E * ceil_div(g.row_tiles * (int64_t)g.columns, kXcds) * kXcds;
    } else {
        blocks = ceil_div(most_row_tiles(T_rows, E, BM) * (int64_t)g.columns, kXcds) * kXcds + (CUT ? kMostCut : 0);
    }
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((gmm_kernel<T, XL, YL, BM, BN, WM, WN, ALIGNED, CUT>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, g);
    return (int)hipGetLastError();
}

template <typename T, int YL, int RT, bool ALIGNED>
int launch_gmm_few(GmmArgs g, int64_t E, int64_t T_rows, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, kFewCols);
    const int64_t blocks = ceil_div(most_row_tiles(T_rows, E, 16 * RT) * (int64_t)g.columns, kXcds) * kXcds;
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((gmm_few_kernel<T, YL, RT, ALIGNED>), dim3((unsigned)blocks), dim3(64 * kFewWaves), 0, s, g);
    return (int)hipGetLastError();
}

template <typename T>
bool chunks_aligned(const void *p, std::initializer_list<int64_t> values) {
    uint64_t bits = reinterpret_cast<uintptr_t>(p);
    for (int64_t v : values) bits |= (uint64_t)(v * (int64_t)sizeof(T));
    return (bits & 15) == 0;
}

// The tile of a rows' product: the least of five estimated times.  The model is fitted to every tile's time on 120 (16-bit) and
// 50 (fp32) random shapes, 1 to 4096 rows per group; its pick is 2.0 % and 2.6 % behind the best tile timed on average
// (38 % and 28 % on the worst shape).  `steps` of 64 bytes of the contraction; `tiles` as if groups were equal, with half a
// tile lost per group.
//   128 x 128, 256 x 256: microseconds a step with one, two, three workgroups on a CU (256 x 256: a quarter, half or
//   whole tile on each CU), by rounds;
//   few rows: a wavefront's chain of units, shared by what a CU holds, or the matrices' bytes at a rate (TB/s).
template <typename T>
int choose_gmm_tile(int64_t T_rows, int64_t E, int64_t N, int64_t K) {
    constexpr bool F32 = sizeof(T) == 4;
    const double mean = (double)T_rows / (double)E, groups = (double)(E < T_rows ? E : T_rows);
    const double steps = (double)ceil_div(K, 64 / (int64_t)sizeof(T));
    auto tiles = [&](int64_t BM, int64_t BN) {
        const double high = mean / (double)BM + 0.5;
        return groups * (high > 1.0 ? high : 1.0) * (double)ceil_div(N, BN);
    };
    auto least = [](double a, double b) { return a < b ? a : b; };
    int best = 1;
    double best_us;
    {
        constexpr double one = F32 ? 0.99 : 0.35, two = F32 ? 2.04 : 0.65, three = F32 ? 3.45 : 1.25, fixed = F32 ? 6.5 : 4.4;
        const double n = tiles(128, 128), rounds = floor(n / 768), rest = n - 768 * rounds;
        best_us = fixed + steps * (rounds * three + (rest <= 0 ? 0 : rest <= 256 ? one : rest <= 512 ? two : three));
    }
    auto consider = [&](int tile, double us) {
        if (us < best_us) best = tile, best_us = us;
    };
    constexpr double kFew[2][3][4] = {{{141, 1.01, 9.0, 6.0}, {147, 1.35, 7.0, 5.8}, {117, 2.07, 3.66, 5.3}},
                                      {{201, 1.70, 7.6, 3.6}, {172, 2.37, 4.7, 4.4}, {135, 3.64, 8.5, 6.8}}};
    for (int i = 0; i < 3; ++i) {
        const double *k = kFew[F32][i], n = tiles(16 << i, kFewCols);
        const double chain = ceil(steps / 16) * k[1] * (n > k[0] ? n / k[0] : 1.0), read = n * steps * 4096e-6 / k[2];
        consider(2 + i, k[3] + (chain > read ? chain : read));
    }
    if constexpr (!F32) {
        const double n = tiles(256, 256), rounds = floor(n / 256), rest = n - 256 * rounds;
        consider(5, 5.3 + steps * (rounds * 1.30 + least(0.90, rest <= 0 ? 0 : rest <= 64 ? 0.31 : rest <= 128 ? 0.55 : 0.90)));
    }
    return best;
}

// The tile of the weights' gradient: 64 x 64 where larger ones would leave CUs idle under long contractions (a matrix of
// 144 x 344 over 3150 rows: 18 us, 24 on 128 x 128), 256 x 256 where there are enough and they pad little (20 of
// 2200 x 1712 over 13120 rows: 150 us, 200 on 128 x 128).  fp32 has four times the MFMA time per step and wants small tiles longer.
template <typename T>
int choose_weights_tile(int64_t E, int64_t K, int64_t N) {
    const int64_t mid = E * ceil_div(K, 128) * ceil_div(N, 128), big = E * ceil_div(K, 256) * ceil_div(N, 256);
    if (mid < (sizeof(T) == 4 ? 1024 : 160)) return 2;
    return sizeof(T) == 2 && big >= 200 && big * 4 <= mid + mid / 7 ? 5 : 1;
}

// x: the rows' operand (a; a transposed for the weights), y: the matrices or g.
template <typename T, int XL, int YL>
int launch_gmm(const GmmArgs &g, int64_t E, int64_t T_rows, int tile, hipStream_t s) {
    const bool aligned = chunks_aligned<T>(g.x, {g.ldx, XL == kInner ? g.K : g.M}) &&
                         chunks_aligned<T>(g.y, {g.ldy, g.y_group, YL == kInner ? g.K : g.N});
    if (tile == 0) tile = XL == kOuter ? choose_weights_tile<T>(E, g.M, g.N) : choose_gmm_tile<T>(T_rows, E, g.N, g.K);
    if constexpr (XL == kInner) {
        switch (tile) {
            case 2: return aligned ? launch_gmm_few<T, YL, 1, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 1, false>(g, E, T_rows, s);
            case 3: return aligned ? launch_gmm_few<T, YL, 2, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 2, false>(g, E, T_rows, s);
            case 4: return aligned ? launch_gmm_few<T, YL, 4, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 4, false>(g, E, T_rows, s);
            default: break;
        }
    } else if (tile == 2) {
        return aligned ? launch_gmm_tile<T, XL, YL, 64, 64, 2, 2, true>(g, E, T_rows, s)
                       : launch_gmm_tile<T, XL, YL, 64, 64, 2, 2, false>(g, E, T_rows, s);
    }
    if constexpr (sizeof(T) == 2) {
        if (tile == 5)  // whose aligned form also writes whole chunks
            return aligned && chunks_aligned<T>(g.out, {g.N}) ? launch_gmm_tile<T, XL, YL, 256, 256, 2, 4, true, XL == kInner>(g, E, T_rows, s)
                           : launch_gmm_tile<T, XL, YL, 256, 256, 2, 4, false, XL == kInner>(g, E, T_rows, s);
    }
    return aligned ? launch_gmm_tile<T, XL, YL, 128, 128, 2, 2, true>(g, E, T_rows, s)
                   : launch_gmm_tile<T, XL, YL, 128, 128, 2, 2, false>(g, E, T_rows, s);
}

template <typename T>
int launch_gmm_type(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, hipStream_t s) {
    if (weights) return launch_gmm<T, kOuter, kOuter>(g, E, T_rows, tile, s);
    return y_inner ? launch_gmm<T, kInner, kInner>(g, E, T_rows, tile, s) : launch_gmm<T, kInner, kOuter>(g, E, T_rows, tile, s);
}

int gmm_bf16(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, hipStream_t s);
int gmm_f16(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, hipStream_t s);
int gmm_f32(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, hipStream_t s);

}  // namespace trt
