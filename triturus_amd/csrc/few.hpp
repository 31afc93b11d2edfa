// Products of ragged groups with few rows each (a decoding batch): bound by reading every matrix once.
//
// A workgroup makes 16 RT rows x 64 columns of one group, and its W wavefronts cut the contraction: no operand is
// shared between wavefronts, so the matrix goes from memory straight into MFMA operands (16 x 16 x 32 of 16 bits,
// 16 x 16 x 4 of fp32) with no barrier before the end, where the W partial tiles meet in LDS in a fixed order.
// A wavefront's unit is 64 bytes of the contraction by 64 columns:
//   INNER (contraction contiguous): lane (n, g) reads the 16 bytes g of column n, 4 times for 4 x 16 columns;
//   OUTER (columns contiguous): lane (c, g) reads, for each of its 16 bytes' worth of contracted values, 4 neighbouring
//          columns (8 bytes of 16-bit types, 16 of fp32); 16-bit values are turned round in registers, 4 byte
//          permutations per 4 columns and pair of rows.
// D units are in flight per wavefront while another is multiplied.  Under 16 rows an INNER matrix is cut into tiles of 32 columns,
// or 16 where those would be fewer than the CUs, with as many more units in flight; an OUTER one among 16 wavefronts there.
// Bound: HBM.  256 rows over 64 groups of 2048 x 1024 (bf16, N x K): 51.8 us, the matrices at 5.2 TB/s; 2 rows of 2 of 8 groups,
// 1024 x 4096: 5.9 us on the GPU, of which an empty launch is 2.9.
#pragma once

#include "gmm.hpp"

namespace trt {

constexpr int kFewCols = 64;  // of a workgroup's usual tile

template <typename T>
struct FewMfma;
template <>
struct FewMfma<__bf16> {
    static __device__ __forceinline__ floatx4 step(uintx4 x, uintx4 y, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    }
};
template <>
struct FewMfma<_Float16> {
    static __device__ __forceinline__ floatx4 step(uintx4 x, uintx4 y, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    }
};
template <>
struct FewMfma<float> {
    static __device__ __forceinline__ floatx4 step(uintx4 x, uintx4 y, floatx4 c) {
        const floatx4 u = __builtin_bit_cast(floatx4, x), v = __builtin_bit_cast(floatx4, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(u[i], v[i], c, 0, 0, 0);
        return c;
    }
};

// LDS of a tile of 16 RT rows and 16 CW columns whose contraction W wavefronts cut.
template <int RT, int CW, int W>
struct FewLds {
    static constexpr int ROW = 16 * CW + 4, PART = 16 * RT * ROW, FLOATS = W * PART;
};

// The wavefronts' parts of a tile, summed in order and written.  acc[i][j][q]: row 16 i + 4 (lane / 16) + q, column
// of(j, lane % 16).
template <typename T, int RT, int CW, int W, typename F>
__device__ __forceinline__ void store_few(const floatx4 (&acc)[RT][CW], float *lds, int wave, T *out, int64_t N, int64_t rows, int64_t cols, F of) {
    constexpr int ROW = FewLds<RT, CW, W>::ROW, PART = FewLds<RT, CW, W>::PART, COLS = 16 * CW;
    const int l = lane_id();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) lds[wave * PART + (16 * i + 4 * (l >> 4) + q) * ROW + of(j, l & 15)] = acc[i][j][q];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * RT * COLS; i += 64 * W) {
        const int r = i / COLS, c = i % COLS;
        if (r >= rows || c >= cols) continue;
        float v = lds[r * ROW + c];
#pragma unroll
        for (int w = 1; w < W; ++w) v += lds[w * PART + r * ROW + c];
        out[(int64_t)r * N + c] = (T)v;
    }
}

template <typename T, int YL, int RT, bool ALIGNED, int CW = 4, int W = 8, int D = 2>
__global__ __launch_bounds__(64 * W) void gmm_few_kernel(GmmArgs g) {
    static_assert(CW == 4 || (YL == kInner && ALIGNED), "4 neighbouring columns of an OUTER matrix are a lane's");
    constexpr int V = 16 / sizeof(T), KT = 64 / sizeof(T);  // values of a chunk, of a unit
    constexpr int COLS = 16 * CW;
    constexpr int CB = 4 * sizeof(T);                       // bytes of a lane's 4 columns (OUTER)
    __shared__ float lds[FewLds<RT, CW, W>::FLOATS];
    GroupTile t;
    if (!find_tile<16 * RT>(g.sizes, blockIdx.x, g.columns, t)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id(), m = l & 15, gk = l >> 4;
    const int64_t col0 = t.column * COLS, rows = t.rows, cols = g.N - col0;
    const int64_t terms = t.group < g.sizes.E ? g.K : 0;  // behind the last group: zeros
    const T *x = static_cast<const T *>(g.x) + t.row0 * g.ldx;
    const T *y = static_cast<const T *>(g.y) + (t.group < g.sizes.E ? t.group : 0) * g.y_group + col0 * (YL == kInner ? g.ldy : 1);

    floatx4 acc[RT][CW];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    struct Unit {
        uintx4 x[RT];
        uintx4 y[CW];  // INNER: CW columns' chunks; OUTER: V rows of CB bytes
    };
    const int64_t units = ceil_div(terms, KT);
    auto load = [&](int64_t u, Unit &n) {
        const int64_t k0 = u * KT, left = terms - k0 - gk * V;  // of the lane's chunk
        const T *xp = x + k0, *yp = y + (YL == kInner ? k0 : k0 * g.ldy);
        if constexpr (ALIGNED) {
            const __amdgpu_buffer_rsrc_t xr = make_rsrc(xp, 0x7fffffff), yr = make_rsrc(yp, 0x7fffffff);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int r = 16 * i + m;
                n.x[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, left > 0 && r < rows ? r * (uint32_t)(g.ldx * sizeof(T)) + gk * 16 : 0x80000000u, 0, 0);
            }
            if constexpr (YL == kInner) {
#pragma unroll
                for (int j = 0; j < CW; ++j) {
                    const int c = 16 * j + m;
                    n.y[j] = __builtin_amdgcn_raw_buffer_load_b128(yr, left > 0 && c < cols ? c * (uint32_t)(g.ldy * sizeof(T)) + gk * 16 : 0x80000000u, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const uint32_t at = i < left && 4 * m < cols ? (gk * V + i) * (uint32_t)(g.ldy * sizeof(T)) + m * CB : 0x80000000u;
                    if constexpr (sizeof(T) == 4) {
                        n.y[i] = __builtin_amdgcn_raw_buffer_load_b128(yr, at, 0, 0);
                    } else {
                        const uintx2 v = __builtin_bit_cast(uintx2, __builtin_amdgcn_raw_buffer_load_b64(yr, at, 0, 0));
                        n.y[i / 2][i % 2 * 2] = v[0], n.y[i / 2][i % 2 * 2 + 1] = v[1];
                    }
                }
            }
        } else if (k0 + KT <= terms && (YL == kInner || cols >= kFewCols)) {
            // every chunk is whole; a row or column that does not exist is read as the last one that does, and never written
            const int rlast = rows < 16 * RT ? (int)rows - 1 : 16 * RT - 1, clast = cols < kFewCols ? (int)cols - 1 : kFewCols - 1;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int r = 16 * i + m < rlast ? 16 * i + m : rlast;
                __builtin_memcpy(&n.x[i], xp + r * g.ldx + gk * V, 16);
            }
#pragma unroll
            for (int i = 0; i < (YL == kInner ? 4 : V); ++i) {
                if constexpr (YL == kInner) {
                    const int c = 16 * i + m < clast ? 16 * i + m : clast;
                    __builtin_memcpy(&n.y[i], yp + c * g.ldy + gk * V, 16);
                } else if constexpr (sizeof(T) == 4) {
                    __builtin_memcpy(&n.y[i], yp + (gk * V + i) * g.ldy + 4 * m, 16);
                } else {
                    uintx2 v;
                    __builtin_memcpy(&v, yp + (gk * V + i) * g.ldy + 4 * m, 8);
                    n.y[i / 2][i % 2 * 2] = v[0], n.y[i / 2][i % 2 * 2 + 1] = v[1];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < RT; ++i) n.x[i] = load_chunk(xp + (16 * i + m) * g.ldx + gk * V, 16 * i + m < rows ? left : 0);
            if constexpr (YL == kInner) {
#pragma unroll
                for (int j = 0; j < 4; ++j) n.y[j] = load_chunk(yp + (16 * j + m) * g.ldy + gk * V, 16 * j + m < cols ? left : 0);
            } else {
                const int64_t in = cols - 4 * m;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const T *p = yp + (gk * V + i) * g.ldy + 4 * m;
                    T e[4] = {T(0), T(0), T(0), T(0)};
                    if (i < left) {
                        if (in >= 4) {
                            __builtin_memcpy(e, p, CB);
                        } else {
#pragma unroll
                            for (int c = 0; c < 3; ++c)
                                if (c < in) e[c] = p[c];
                        }
                    }
                    if constexpr (sizeof(T) == 4) {
                        __builtin_memcpy(&n.y[i], e, 16);
                    } else {
                        uintx2 v;
                        __builtin_memcpy(&v, e, 8);
                        n.y[i / 2][i % 2 * 2] = v[0], n.y[i / 2][i % 2 * 2 + 1] = v[1];
                    }
                }
            }
        }
    };
    auto multiply = [&](const Unit &n) {
        uintx4 f[CW];  // columns' chunks
        if constexpr (YL == kInner) {
#pragma unroll
            for (int j = 0; j < CW; ++j) f[j] = n.y[j];
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = uintx4{n.y[0][j], n.y[1][j], n.y[2][j], n.y[3][j]};
        } else {
#pragma unroll
            for (int p = 0; p < 4; ++p) {  // rows 2 p and 2 p + 1: words {c0 c1}, {c2 c3} of each
                f[0][p] = __builtin_amdgcn_perm(n.y[p][2], n.y[p][0], 0x05040100);
                f[1][p] = __builtin_amdgcn_perm(n.y[p][2], n.y[p][0], 0x07060302);
                f[2][p] = __builtin_amdgcn_perm(n.y[p][3], n.y[p][1], 0x05040100);
                f[3][p] = __builtin_amdgcn_perm(n.y[p][3], n.y[p][1], 0x07060302);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < CW; ++j) acc[i][j] = FewMfma<T>::step(n.x[i], f[j], acc[i][j]);
    };
    int64_t u = D * wave;  // neighbours: together whole 128-byte lines of an INNER matrix
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
    store_few<T, RT, CW, W>(acc, lds, wave, static_cast<T *>(g.out) + t.row0 * g.N + col0, g.N, rows, cols,
                            [](int j, int c) { return YL == kInner ? 16 * j + c : 4 * c + j; });
}

}  // namespace trt
