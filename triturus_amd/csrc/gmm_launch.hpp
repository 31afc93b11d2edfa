// The choice of a tile for a product of ragged groups, shared by the element types.
#pragma once

#include <initializer_list>

#include "few.hpp"
#include "tile_cost.hpp"

namespace trt {

inline int64_t most_pieces(int64_t T, int64_t E, int64_t len) { return T / len + (E < T ? E : T); }

// Tiles of the rows' products: 1 = 128 x 128, 2, 3, 4 = 16, 32, 64 rows x 64 columns of the few-row kernel, 5 = 256 x 256
// (16-bit types) or 64 x 64 (fp32).  Of the weights' gradient: 1 = 128 x 128, 2 = 64 x 64, 5 = 256 x 256.
template <typename T, int XL, int YL, int BM, int BN, int WM, int WN, bool ALIGNED, bool CUT = false>
int launch_gmm_tile(GmmArgs g, int64_t E, int64_t T_rows, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, BN);
    int64_t blocks;
    if (XL == kOuter) {
        g.row_tiles = (uint32_t)ceil_div(g.M, BM);
        const bool cut = BM == 128 && g.partial;
        if (!cut) g.piece = {};
        blocks = (cut ? most_pieces(T_rows, E, g.piece.d) : E) * ceil_div(g.row_tiles * (int64_t)g.columns, kXcds) * kXcds;
    } else {
        blocks = ceil_div(most_row_tiles(T_rows, E, BM) * (int64_t)g.columns, kXcds) * kXcds + (CUT ? kMostCut : 0);
    }
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((gmm_kernel<T, XL, YL, BM, BN, WM, WN, ALIGNED, CUT>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, g);
    return (int)hipGetLastError();
}

template <typename T, int YL, int RT, bool ALIGNED, int CW = 4, int W = 8, int D = 2>
int launch_gmm_few(GmmArgs g, int64_t E, int64_t T_rows, hipStream_t s) {
    g.columns = (uint32_t)ceil_div(g.N, 16 * CW);
    const int64_t blocks = ceil_div(most_row_tiles(T_rows, E, 16 * RT) * (int64_t)g.columns, kXcds) * kXcds;
    if (blocks >= (int64_t)1 << 31) return TRT_E_RANGE;
    hipLaunchKernelGGL((gmm_few_kernel<T, YL, RT, ALIGNED, CW, W, D>), dim3((unsigned)blocks), dim3(64 * W), 0, s, g);
    return (int)hipGetLastError();
}

// 16 rows a tile: more and smaller pieces where there are fewer tiles than CUs.  An INNER matrix is always read in tiles of
// 32 columns or fewer: a wavefront's 4 units are then 256 neighbouring bytes of a column, whole pairs of lines (64 rows
// of 8 groups, 4096 x 4096 bf16: 72.2 us with 64 columns and 2 units, 63.9 us so; 256 rows of 64, 2048 x 1024: 53.8 -> 51.6 us).
template <typename T, int YL>
int launch_gmm_few_rows(const GmmArgs &g, int64_t E, int64_t T_rows, hipStream_t s) {
    const double n = GroupedShape(T_rows, E, g.N, 64).tiles(16, kFewCols);
    if constexpr (YL == kInner) {
        if (n <= 64) return launch_gmm_few<T, YL, 1, true, 1, 8, 8>(g, E, T_rows, s);
        return launch_gmm_few<T, YL, 1, true, 2, 8, 4>(g, E, T_rows, s);
    } else if (n <= 256) {
        return launch_gmm_few<T, YL, 1, true, 4, 16, 2>(g, E, T_rows, s);
    } else {
        return launch_gmm_few<T, YL, 1, true>(g, E, T_rows, s);
    }
}

template <typename T>
bool chunks_aligned(const void *p, std::initializer_list<int64_t> values) {
    uint64_t bits = reinterpret_cast<uintptr_t>(p);
    for (int64_t v : values) bits |= (uint64_t)(v * (int64_t)sizeof(T));
    return (bits & 15) == 0;
}

// The tile of a rows' product: the least of the estimated times (tile_cost.hpp).
template <typename T>
int choose_gmm_tile(int64_t T_rows, int64_t E, int64_t N, int64_t K, bool y_inner, double *us = nullptr) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr MidCost kMid = F32 ? MidCost{0.980, 1.98, 2.91, 2.4, 11.4} : MidCost{0.317, 0.440, 1.058, 5.3, 2.0};
    constexpr BigCost kBig = {0.824, 0.459, 0.276, 3.5, 4.6};
    constexpr SmallCost kSmall = {0.340, 0.293, 4.5};  // fp32
    constexpr FewCost kFew[2][3] = {{{149, 1.09, 8.0, 5.4}, {147, 1.30, 6.8, 5.9}, {112, 1.80, 5.2, 6.4}},
                                    {{143, 0.77, 9.5, 5.9}, {185, 1.89, 5.3, 5.3}, {167, 3.73, 2.7, 5.4}}};
    const GroupedShape g(T_rows, E, N, K * (int64_t)sizeof(T));
    auto least = [&](double us, double inner, double outer) {  // not below the matrices' reading
        const double read = g.stream(y_inner ? inner : outer);
        return us > read ? us : read;
    };
    int best = 1;
    double best_us = least(estimate(g, kMid), 4.2, 5.4);
    auto consider = [&](int tile, double us) {
        if (us < best_us) best = tile, best_us = us;
    };
    for (int i = 0; i < 3; ++i) consider(2 + i, least(estimate(g, kFew[F32][i], 1 << i), 4.8, 5.2));
    consider(5, least(F32 ? estimate(g, kSmall) : estimate(g, kBig), 4.2, 5.4));
    if (us) *us = best_us;
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

// Into pieces of how many rows the groups are cut, on 128 x 128 tiles, where few tiles have long contractions; 0: not.  `tile`: the
// choice above.  The pieces' sums are added in order by another launch.  Estimates in microseconds, fitted to pieces of a
// 1/32 .. 1 of the mean group on 90 random shapes: a step of 64 bytes a row with up to one, two or more workgroups on a CU, both
// launches, a piece's tile written and read, and without pieces how much longer the longest of several groups is than their mean.
// That is charged for up to one step of a full CU, two where more than 64 groups are taken as they come: beyond it the tiles come in
// rounds, over which long and short groups average out (8 groups of 2048 rows, 2056 x 2048 of fp32: 1077 us whole, 1213 in pieces;
// 9 of 674, 616 x 3000 of bf16: 36 and 72).  The pieces' sums may take 256 MiB, or half of what operands and result take.
// More than 32 pieces of a group are of 1024 rows or more, and pay for the chain of their sums (479454 rows in 2 groups, 88 x 8 of
// fp32: 912 us in pieces of 7520 rows, 497 of 1984; 78 shapes of more than 32768 rows a group: 17 -> 10 % behind the best pieces).
// On 920 random shapes, up to 6000 tiles and 4 million rows, the choice is 6 % behind the best pieces on average and 2.9 times on the
// worst, whole groups 1.6 and 31 times (16384 rows, 512 x 512 of bf16: 175 us, 27 in pieces; 16 uneven groups, 256 x 512: 48 and 26).
constexpr double kMostSums = 256 << 20;
template <typename T>
int64_t choose_weights_piece(int64_t T_rows, int64_t E, int64_t K, int64_t N, int tile) {
    constexpr bool F32 = sizeof(T) == 4;
    if (tile == 5) return 0;
    const double matrix = (double)(ceil_div(K, 128) * ceil_div(N, 128)), mid = (double)E * matrix;
    const double small = ceil((double)E * (double)(ceil_div(K, 64) * ceil_div(N, 64)) / 256), longest = 1.0 + (F32 ? 0.26 : 0.50) * log2((double)(E < 16 ? E : 16));
    constexpr double one = F32 ? 1.05 : 0.36, two = F32 ? 1.93 : 0.57, three = F32 ? 2.79 : 0.855;
    auto step = [](double workgroups) { return workgroups <= 256 ? one : workgroups <= 512 ? two : three * ceil(workgroups / 256) / 3; };
    auto larger = [](double a, double b) { return a > b ? a : b; };
    const double steps = (double)ceil_div(ceil_div(T_rows, E) * (int64_t)sizeof(T), 64);
    const double mean = tile == 2 ? larger(F32 ? 0.382 : 0.314, (F32 ? 0.22 : 0.122) * small) : step(mid);
    const double held = ((double)T_rows * (double)(K + N) + (double)E * (double)K * (double)N) * (double)sizeof(T);
    const double full = E <= kWave ? three : 2 * three;
    double best = 0.97 * (3.3 + steps * larger(mean, longest * (mean < full ? mean : full)));
    int64_t rows = 0;
    for (int64_t p = 1; p <= 2048; p += p < 32 ? 1 : p / 8) {
        const int64_t len = ceil_div(ceil_div(T_rows, E * p), 32) * 32;
        if (len * (int64_t)sizeof(T) < 4 * 64 || (p > 32 && len < 1024)) break;
        if ((double)most_pieces(T_rows, E, len) * matrix * (128 * 128 * sizeof(float)) > larger(kMostSums, 0.5 * held)) break;
        const double n = E == 1 ? (double)ceil_div(T_rows, len) : (double)(T_rows / len) + 0.5 * (double)E, w = n * matrix;
        const double us = (F32 ? 13.3 : 11.5) + (double)(len * (int64_t)sizeof(T) / 64) * step(w) + w * 0.024 + (p > 32 ? 0.25 * (double)p : 0.0);
        if (us < best) best = us, rows = len;
    }
    return rows;
}

// ---- operands off the 16-byte boundaries -------------------------------------------------------------------------------
// Rows that start off them, or are not whole chunks, cost up to twice a product's time (16-byte loads from any address, and no
// loads to LDS), least where both operands lie along the contraction, and the weights' gradient two to three times.  Where that
// is more than a copy, an operand is first copied into rows of whole chunks with zeros behind (16384 rows in 8 groups of fp16,
// K = 2049, N = 2047: 336 us as they are and 205 with both copied; matrices stored N x K 261 and 225; the weights' gradient
// 500 and 191.  On the boundaries they take 157 to 180).

// Rows of n values, `rows` to a group, strides in values, to dense rows of whole chunks.
struct PadJob {
    const void *from;
    void *to;
    int64_t n, ld, group;
    Divider chunks, rows;  // of a row, of a group
    uint32_t total;        // chunks in all
};
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadJob a, PadJob b, PadJob c, uint32_t a_blocks, uint32_t ab_blocks) {
    const PadJob &j = blockIdx.x < a_blocks ? a : blockIdx.x < ab_blocks ? b : c;
    const uint32_t i = (blockIdx.x - (blockIdx.x < a_blocks ? 0 : blockIdx.x < ab_blocks ? a_blocks : ab_blocks)) * 256 + threadIdx.x;
    if (i >= j.total) return;
    constexpr int V = 16 / sizeof(T);
    const uint32_t row = divide(i, j.chunks), at = (i - row * j.chunks.d) * V, e = divide(row, j.rows);
    const T *p = static_cast<const T *>(j.from) + e * j.group + (row - e * j.rows.d) * j.ld + at;
    static_cast<uintx4 *>(j.to)[i] = load_chunk(p, j.n - at);
}

struct PadPlan {
    bool x, y;
    size_t bytes;  // of workspace
};

// us: the product's estimated time on aligned operands; worth: how much of it more the others cost.
template <typename T, int XL, int YL>
PadPlan plan_pads(const GmmArgs &g, int64_t E, int64_t T_rows, double us, double worth) {
    constexpr int64_t V = 16 / sizeof(T);
    const int64_t xn = XL == kInner ? g.K : g.M, yn = YL == kInner ? g.K : g.N, yrows = XL == kOuter ? T_rows : YL == kInner ? E * g.N : E * g.K;
    PadPlan p = {!chunks_aligned<T>(g.x, {g.ldx, xn}), !chunks_aligned<T>(g.y, {g.ldy, g.y_group, yn}), 0};
    const int64_t x_chunks = p.x ? T_rows * ceil_div(xn, V) : 0, y_chunks = p.y ? yrows * ceil_div(yn, V) : 0;
    const double copy = 4.0 + (double)(x_chunks + y_chunks) * 32e-6 / 4.5;
    if (x_chunks >= (int64_t)1 << 30 || y_chunks >= (int64_t)1 << 30 || copy > worth * us) return {false, false, 0};
    p.bytes = (size_t)(x_chunks + y_chunks) * 16;
    return p;
}

// A copy of `groups` matrices to `to`, which moves on behind it; from, ld and group become the copy's.
template <typename T>
PadJob pad_job(bool wanted, const void *&from, int64_t &ld, int64_t *group, int64_t n, int64_t rows, int64_t groups, char *&to) {
    PadJob j = {};
    if (!wanted) return j;
    constexpr int64_t V = 16 / sizeof(T);
    const int64_t chunks = ceil_div(n, V);
    j = {from, to, n, ld, group ? *group : 0, divider((uint32_t)chunks), divider((uint32_t)rows), (uint32_t)(groups * rows * chunks)};
    from = to;
    to += (size_t)j.total * 16;
    ld = chunks * V;
    if (group) *group = rows * ld;
    return j;
}
// The rows' operand or, of a rows' product, the matrices.
template <typename T, int XL>
PadJob pad_x(bool wanted, GmmArgs &g, int64_t T_rows, char *&to) {
    return pad_job<T>(wanted, g.x, g.ldx, nullptr, XL == kInner ? g.K : g.M, T_rows, 1, to);
}
template <typename T, int XL, int YL>
PadJob pad_y(bool wanted, GmmArgs &g, int64_t E, int64_t T_rows, char *&to) {
    if (XL == kOuter) return pad_job<T>(wanted, g.y, g.ldy, nullptr, g.N, T_rows, 1, to);
    return pad_job<T>(wanted, g.y, g.ldy, &g.y_group, YL == kInner ? g.K : g.N, YL == kInner ? g.N : g.K, E, to);
}
template <typename T>
int launch_pads(const PadJob &a, const PadJob &b, const PadJob &c, hipStream_t s) {
    const uint32_t a_blocks = (uint32_t)ceil_div(a.total, 256), ab = a_blocks + (uint32_t)ceil_div(b.total, 256), all = ab + (uint32_t)ceil_div(c.total, 256);
    hipLaunchKernelGGL(pad_rows_kernel<T>, dim3(all), dim3(256), 0, s, a, b, c, a_blocks, ab);
    return (int)hipGetLastError();
}

struct Workspace {
    void *p;
    size_t bytes;
    size_t *query;  // not null: only say how many are wanted
};

// How a product is made: its tile, the rows of a piece (0: groups are whole), the copies, and the bytes of the pieces' sums.
struct GmmPlan {
    int tile;
    int64_t piece;
    PadPlan pads;
    size_t partial;
};

// x: the rows' operand (a; a transposed for the weights), y: the matrices or g.
template <typename T, int XL, int YL>
GmmPlan plan_gmm(const GmmArgs &g, int64_t E, int64_t T_rows, int tile) {
    GmmPlan p = {tile, 0, {false, false, 0}, 0};
    double us = 0.0;
    if constexpr (XL == kOuter) {
        if (tile == 0) {
            p.tile = choose_weights_tile<T>(E, g.M, g.N);
            p.piece = choose_weights_piece<T>(T_rows, E, g.M, g.N, p.tile);
        }
        us = 10.0 + 2.0 * (double)T_rows * (double)g.M * (double)g.N / (sizeof(T) == 4 ? 60e6 : 900e6);
    } else {
        const int best = choose_gmm_tile<T>(T_rows, E, g.N, g.K, YL == kInner, &us);
        if (tile == 0) p.tile = best;
    }
    // few rows are bound by reading the matrices, and a copy reads and writes them
    const bool few = XL == kInner && p.tile >= 2 && p.tile <= 4;
    if (!few) p.pads = plan_pads<T, XL, YL>(g, E, T_rows, us, XL == kOuter ? 1.2 : YL == kOuter ? 0.8 : 0.5);
    if (p.piece) p.partial = (size_t)(most_pieces(T_rows, E, p.piece) * ceil_div(g.M, 128) * ceil_div(g.N, 128)) * (128 * 128 * sizeof(float));
    return p;
}

template <typename T, int XL>
bool x_aligned(const GmmArgs &g) { return chunks_aligned<T>(g.x, {g.ldx, XL == kInner ? g.K : g.M}); }
template <typename T, int YL>
bool y_aligned(const GmmArgs &g) { return chunks_aligned<T>(g.y, {g.ldy, g.y_group, YL == kInner ? g.K : g.N}); }

// aligned: both operands' rows are whole chunks on their boundaries.
template <typename T, int XL, int YL>
int run_gmm(GmmArgs g, int64_t E, int64_t T_rows, int tile, bool aligned, hipStream_t s) {
    if (g.partial) tile = 1;
    if constexpr (XL == kInner) {
        switch (tile) {
            case 2: return aligned ? launch_gmm_few_rows<T, YL>(g, E, T_rows, s) : launch_gmm_few<T, YL, 1, false>(g, E, T_rows, s);
            case 3: return aligned ? launch_gmm_few<T, YL, 2, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 2, false>(g, E, T_rows, s);
            case 4: return aligned ? launch_gmm_few<T, YL, 4, true>(g, E, T_rows, s) : launch_gmm_few<T, YL, 4, false>(g, E, T_rows, s);
            default: break;
        }
    } else if (tile == 2) {
        return aligned ? launch_gmm_tile<T, XL, YL, 64, 64, 2, 2, true>(g, E, T_rows, s)
                       : launch_gmm_tile<T, XL, YL, 64, 64, 2, 2, false>(g, E, T_rows, s);
    }
    if constexpr (sizeof(T) == 2) {
        if (tile == 5)
            return aligned ? launch_gmm_tile<T, XL, YL, 256, 256, 2, 4, true, XL == kInner>(g, E, T_rows, s)
                           : launch_gmm_tile<T, XL, YL, 256, 256, 2, 4, false, XL == kInner>(g, E, T_rows, s);
    } else if constexpr (XL == kInner) {
        if (tile == 5)
            return aligned ? launch_gmm_tile<T, XL, YL, 64, 64, 2, 2, true>(g, E, T_rows, s)
                           : launch_gmm_tile<T, XL, YL, 64, 64, 2, 2, false>(g, E, T_rows, s);
    }
    const int status = aligned ? launch_gmm_tile<T, XL, YL, 128, 128, 2, 2, true>(g, E, T_rows, s)
                               : launch_gmm_tile<T, XL, YL, 128, 128, 2, 2, false>(g, E, T_rows, s);
    if constexpr (XL == kOuter) {
        if (!status && g.partial) {
            g.row_tiles = (uint32_t)ceil_div(g.M, 128), g.columns = (uint32_t)ceil_div(g.N, 128);
            const int64_t blocks = E * g.row_tiles * g.columns * 8;
            hipLaunchKernelGGL(gmm_join_kernel<T>, dim3((unsigned)blocks), dim3(kWave), 0, s, g);
            return (int)hipGetLastError();
        }
    }
    return status;
}

template <typename T, int XL, int YL>
int launch_gmm(GmmArgs g, int64_t E, int64_t T_rows, int tile, const Workspace &w, hipStream_t s) {
    const GmmPlan p = plan_gmm<T, XL, YL>(g, E, T_rows, tile);
    if (w.query) {
        *w.query = p.pads.bytes + p.partial;
        return TRT_OK;
    }
    bool aligned = x_aligned<T, XL>(g) && y_aligned<T, YL>(g);
    if (w.p && w.bytes >= p.pads.bytes + p.partial) {  // without a workspace operands are read as they are, and groups not cut
        char *to = static_cast<char *>(w.p);
        if (p.pads.bytes) {
            const PadJob x = pad_x<T, XL>(p.pads.x, g, T_rows, to), y = pad_y<T, XL, YL>(p.pads.y, g, E, T_rows, to);
            const int status = launch_pads<T>(x, y, {}, s);
            if (status) return status;
            aligned = true;
        }
        if (p.partial) g.partial = reinterpret_cast<float *>(to), g.piece = divider((uint32_t)p.piece);
    }
    return run_gmm<T, XL, YL>(g, E, T_rows, p.tile, aligned, s);
}

// Both gradients: r is a's (its x is g), w the matrices' (its y is g).  g is copied once for both, and all copies are one launch.
template <typename T, int YL>
int launch_gmm_grad(GmmArgs r, GmmArgs w, int64_t E, int64_t T_rows, const Workspace &ws, hipStream_t s) {
    const GmmPlan pr = plan_gmm<T, kInner, YL>(r, E, T_rows, 0), pw = plan_gmm<T, kOuter, kOuter>(w, E, T_rows, 0);
    const bool pad_g = pr.pads.x || pw.pads.y;
    bool g_ok = x_aligned<T, kInner>(r), b_ok = y_aligned<T, YL>(r), a_ok = x_aligned<T, kOuter>(w);
    GmmArgs rp = r, wp = w;
    char *const base = static_cast<char *>(ws.p), *to = base;
    const PadJob g = pad_x<T, kInner>(pad_g, rp, T_rows, to), b = pad_y<T, kInner, YL>(pr.pads.y, rp, E, T_rows, to), a = pad_x<T, kOuter>(pw.pads.x, wp, T_rows, to);
    const size_t copies = (size_t)g.total * 16 + (size_t)b.total * 16 + (size_t)a.total * 16;
    if (ws.query) {
        *ws.query = copies + pw.partial;
        return TRT_OK;
    }
    if (ws.p && ws.bytes >= copies + pw.partial) {
        if (pad_g) wp.y = rp.x, wp.ldy = rp.ldx;
        r = rp, w = wp;
        if (copies) {
            const int status = launch_pads<T>(g, b, a, s);
            if (status) return status;
            g_ok = g_ok || pad_g, b_ok = b_ok || pr.pads.y, a_ok = a_ok || pw.pads.x;
        }
        if (pw.partial) w.partial = reinterpret_cast<float *>(base + copies), w.piece = divider((uint32_t)pw.piece);
    }
    const int status = run_gmm<T, kInner, YL>(r, E, T_rows, pr.tile, g_ok && b_ok, s);
    return status ? status : run_gmm<T, kOuter, kOuter>(w, E, T_rows, pw.tile, a_ok && g_ok, s);
}

template <typename T>
int launch_gmm_grad_type(const GmmArgs &r, const GmmArgs &w, int64_t E, int64_t T_rows, bool y_inner, const Workspace &ws, hipStream_t s) {
    return y_inner ? launch_gmm_grad<T, kInner>(r, w, E, T_rows, ws, s) : launch_gmm_grad<T, kOuter>(r, w, E, T_rows, ws, s);
}

template <typename T>
int launch_gmm_type(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s) {
    if (weights) return launch_gmm<T, kOuter, kOuter>(g, E, T_rows, tile, w, s);
    return y_inner ? launch_gmm<T, kInner, kInner>(g, E, T_rows, tile, w, s) : launch_gmm<T, kInner, kOuter>(g, E, T_rows, tile, w, s);
}

int gmm_bf16(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s);
int gmm_f16(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s);
int gmm_f32(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s);

int gmm_grad_bf16(const GmmArgs &r, const GmmArgs &w, int64_t E, int64_t T_rows, bool y_inner, const Workspace &ws, hipStream_t s);
int gmm_grad_f16(const GmmArgs &r, const GmmArgs &w, int64_t E, int64_t T_rows, bool y_inner, const Workspace &ws, hipStream_t s);
int gmm_grad_f32(const GmmArgs &r, const GmmArgs &w, int64_t E, int64_t T_rows, bool y_inner, const Workspace &ws, hipStream_t s);

}  // namespace trt
