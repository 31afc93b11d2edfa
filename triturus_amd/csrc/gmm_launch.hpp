// The choice of a tile for a product of ragged groups, shared by the element types.
#pragma once

#include "few.hpp"

namespace trt {

// Tiles: 1 = 128 x 128 (4 wavefronts), 2, 3, 4 = 16, 32, 64 rows x 64 columns of the few-row kernel.
template <typename T, int XL, int YL, int BM, int BN, int WM, int WN, bool ALIGNED>
int launch_gmm_tile(GmmArgs g, int64_t E, int64_t T_rows, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, BN);
    int64_t blocks;
    if (XL == kOuter) {
        g.row_tiles = (uint32_t)ceil_div(g.M, BM);
        blocks = ceil_div(E * g.row_tiles * (int64_t)g.columns, kXcds) * kXcds;
    } else {
        blocks = ceil_div(most_row_tiles(T_rows, E, BM) * (int64_t)g.columns, kXcds) * kXcds;
    }
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((gmm_kernel<T, XL, YL, BM, BN, WM, WN, ALIGNED>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, g);
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

// x: the rows' operand (a; a transposed for the weights), y: the matrices or g.
template <typename T, int XL, int YL>
int launch_gmm(const GmmArgs &g, int64_t E, int64_t T_rows, int tile, hipStream_t s) {
    const bool aligned = chunks_aligned<T>(g.x, {g.ldx, XL == kInner ? g.K : g.M}) &&
                         chunks_aligned<T>(g.y, {g.ldy, g.y_group, YL == kInner ? g.K : g.N});
    if constexpr (XL == kInner) {
        if (tile == 0) {
            const int64_t mean = T_rows / E;
            tile = mean <= 16 ? 2 : mean <= 32 ? 3 : mean <= 64 ? 4 : 1;
        }
        switch (tile) {
            case 2: return aligned ? launch_gmm_few<T, YL, 1, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 1, false>(g, E, T_rows, s);
            case 3: return aligned ? launch_gmm_few<T, YL, 2, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 2, false>(g, E, T_rows, s);
            case 4: return aligned ? launch_gmm_few<T, YL, 4, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 4, false>(g, E, T_rows, s);
            default: break;
        }
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
