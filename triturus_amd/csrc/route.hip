// The router of a mixture layer: the k largest of a row's E logits, their softmax weights, and the chosen pairs
// (row, choice) ordered by expert.
//
// Choosing.  16 lanes hold a row (4 rows a wavefront), V values each, lane by lane in order.  Values become whole
// numbers that compare like them; k times the row's largest is found in 4 lane rotations (DPP, within the 16) and
// the first lane that holds it gives it up -- equal values go to the lowest index.
//
// Ordering is a counting sort, stable in row order and without atomics whose order could matter.  A workgroup has 64
// rows; every expert has a 64-bit mask of the rows that chose it (a row chooses an expert at most once), so a
// pair's place among the workgroup's is a population count of the bits below its row.  One workgroup does it all in one
// launch; otherwise the first launch leaves the counts (a byte per expert and workgroup) and the last one adds up what
// stands before it -- by itself up to kDirect workgroups, from a prefix sum made by a launch between them above that.
// Bound: launches and latency for small T (64 rows of 64: 3.3 us).  For large T the choice: 65536 rows of 128 fp32 logits take 8.5 us
// (3.9 TB/s) and 1.2 to 1.4 more for each of the k choices, some 50 vector instructions; then 4.8 us for the sums, 7 for the places.
#include "grouped.hpp"

namespace trt {

constexpr int kRouteRows = 64;   // of a workgroup
constexpr int kRouteMost = 16;   // choices: one lane of a row's 16 each
constexpr int kRouteExperts = 1024;
constexpr int kDirect = 64;      // workgroups whose counts the last launch adds up by itself

struct RouteArgs {
    const void *logits;
    float *weights;
    int32_t *experts, *rows, *slots, *sizes;
    uint8_t *counts;   // [expert][pitch], a byte per workgroup
    uint32_t *before;  // [expert][pitch]: pairs of the expert in the workgroups before (above kDirect workgroups)
    int64_t T, ld, pitch;
    int E, k, normalize;
};

template <int CTRL>
__device__ __forceinline__ uint32_t rotate16(uint32_t v) {
    return __builtin_amdgcn_mov_dpp(v, 0x120 + CTRL, 0xf, 0xf, true);  // row_ror
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    uint32_t u;
    u = rotate16<8>(v), v = u > v ? u : v;
    u = rotate16<4>(v), v = u > v ? u : v;
    u = rotate16<2>(v), v = u > v ? u : v;
    u = rotate16<1>(v), v = u > v ? u : v;
    return v;
}
__device__ __forceinline__ float row_sum(float v) {
    v += __builtin_bit_cast(float, rotate16<8>(__builtin_bit_cast(uint32_t, v)));
    v += __builtin_bit_cast(float, rotate16<4>(__builtin_bit_cast(uint32_t, v)));
    v += __builtin_bit_cast(float, rotate16<2>(__builtin_bit_cast(uint32_t, v)));
    v += __builtin_bit_cast(float, rotate16<1>(__builtin_bit_cast(uint32_t, v)));
    return v;
}

// Whole numbers in the order of the values, -0 as 0 and NaN above everything; up to kNever: -inf, never chosen.
constexpr uint32_t kNever = 0x007fffffu;
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x != x ? __builtin_nanf("") : x + 0.0f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The lane's V logits of a row, -inf where there is none.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T *row, int lane, int64_t E, float (&x)[V]) {
    constexpr int C = 16 / sizeof(T);
    if constexpr (V >= C) {
#pragma unroll
        for (int i = 0; i < V / C; ++i) {
            const int64_t at = lane * V + i * C, left = E - at;
            const uintx4 u = load_chunk(row + at, left);
            T e[C];
            __builtin_memcpy(e, &u, 16);
#pragma unroll
            for (int j = 0; j < C; ++j) x[i * C + j] = j < left ? (float)e[j] : -__builtin_inff();
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = lane * V + i < E ? (float)row[lane * V + i] : -__builtin_inff();
    }
}

// Marks a pair in its expert's mask; the result does not depend on the order of the calls.
__device__ __forceinline__ void set_bit(uint64_t *mask, int row) {
    __hip_atomic_fetch_or(mask, (uint64_t)1 << row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// First place of every expert, over all workgroups: `first` holds the counts and becomes their exclusive prefix sum;
// returns the sum.  `part` has a slot per wavefront.
template <int THREADS>
__device__ __forceinline__ uint32_t prefix_experts(uint32_t *first, int E, uint32_t *part) {
    uint32_t before = 0;
    const int tid = threadIdx.x, w = tid / kWave;
    for (int e0 = 0; e0 < E; e0 += THREADS) {
        const int e = e0 + tid;
        const uint32_t n = e < E ? first[e] : 0, incl = wave_prefix(n);
        if (lane_id() == kWave - 1) part[w] = incl;
        __syncthreads();
        uint32_t add = before, all = 0;
#pragma unroll
        for (int i = 0; i < THREADS / kWave; ++i) {
            if (i < w) add += part[i];
            all += part[i];
        }
        if (e < E) first[e] = add + incl - n;
        before += all;
        __syncthreads();
    }
    return before;
}

// Writes the pairs of the workgroup's rows: `first[e]` is the place of the expert's first pair in this workgroup.
template <int THREADS>
__device__ __forceinline__ void place_pairs(const RouteArgs &g, int64_t row0, const uint64_t *mask, const uint32_t *first,
                                            const int32_t *chosen, uint32_t total) {
    const int64_t rows = g.T - row0 < kRouteRows ? g.T - row0 : kRouteRows;
    for (int i = threadIdx.x; i < rows * g.k; i += THREADS) {
        const int32_t e = chosen[i];
        const int row = i / g.k;
        int32_t slot = -1;
        if (e >= 0) {
            slot = first[e] + __builtin_popcountll(mask[e] & (((uint64_t)1 << row) - 1));
            g.rows[slot] = (int32_t)(row0 + row);
        }
        g.slots[row0 * g.k + i] = slot;
        if (row0 * g.k + i >= total) g.rows[row0 * g.k + i] = 0;  // places that no pair has
    }
}

// V * 16 >= E.  ONE: a single workgroup, which also orders the pairs.
// 16 wavefronts take all 64 rows at once (a choice is a chain of dependent steps); 4 where a lane's 64 logits leave no
// registers for more.
template <int V>
constexpr int kChooseThreads = V > 32 ? 256 : 1024;

template <typename T, int V, bool ONE>
__global__ __launch_bounds__(kChooseThreads<V>) void route_choose_kernel(RouteArgs g) {
    constexpr int THREADS = kChooseThreads<V>;
    __shared__ uint64_t mask[V * 16];
    __shared__ int32_t chosen[ONE ? kRouteRows * kRouteMost : 1];
    __shared__ uint32_t first[ONE ? V * 16 : 1], part[THREADS / kWave];
    for (int e = threadIdx.x; e < g.E; e += THREADS) mask[e] = 0;
    __syncthreads();
    const int lane = threadIdx.x & 15, shift = lane_id() & 48;
    const int64_t row0 = (int64_t)blockIdx.x * kRouteRows;
    for (int r = threadIdx.x / 16; r < kRouteRows; r += THREADS / 16) {
        const int64_t t = row0 + r;
        if (t >= g.T) break;  // whole rows of 16 lanes
        float x[V];
        load_logits(static_cast<const T *>(g.logits) + t * g.ld, lane, g.E, x);
        uint32_t key[V];
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = order_key(x[i]);
        uint32_t mine = 0;  // lane j: choice j
        int32_t expert = -1;
        float top = 0.0f;
        for (int j = 0; j < g.k; ++j) {
            uint32_t best = key[0];
#pragma unroll
            for (int i = 1; i < V; ++i) best = key[i] > best ? key[i] : best;
            const uint32_t all = row_max(best);
            int at = 0;  // the first place of it
#pragma unroll
            for (int i = V - 1; i >= 0; --i) at = key[i] == all ? i : at;
            const uint32_t holders = (uint32_t)(__ballot(best == all) >> shift) & 0xffff;
            const int winner = __builtin_ctz(holders);
            const int32_t index = __shfl(lane * V + at, shift + winner, kWave);
            if (j == 0) top = key_value(all);
            if (all > kNever && lane == j) mine = all, expert = index;
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = lane == winner && i == at ? 0 : key[i];
        }
        const float e = expert >= 0 ? expf(key_value(mine) - top) : 0.0f;
        float total;
        if (g.normalize) {
            total = row_sum(e);
        } else {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) s += x[i] == -__builtin_inff() ? 0.0f : expf(x[i] - top);
            total = row_sum(s);
        }
        if (lane < g.k) {
            g.weights[t * g.k + lane] = expert >= 0 ? e / total : 0.0f;
            g.experts[t * g.k + lane] = expert;
            if (ONE) chosen[r * g.k + lane] = expert;
            if (expert >= 0) set_bit(&mask[expert], r);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < g.E; e += THREADS) {
        const uint32_t n = __builtin_popcountll(mask[e]);
        if constexpr (ONE) {
            g.sizes[e] = (int32_t)n;
            first[e] = n;
        } else {
            g.counts[e * g.pitch + blockIdx.x] = (uint8_t)n;
        }
    }
    if constexpr (ONE) {
        __syncthreads();
        const uint32_t total = prefix_experts<THREADS>(first, g.E, part);
        place_pairs<THREADS>(g, row0, mask, first, chosen, total);
    }
}

// One workgroup per expert: counts to the sums before each workgroup, and the expert's size.
__global__ __launch_bounds__(256) void route_prefix_kernel(RouteArgs g, int64_t workgroups) {
    __shared__ uint32_t part[4];
    const int w = threadIdx.x / kWave;
    const uint8_t *counts = g.counts + blockIdx.x * g.pitch;
    uint32_t *out = g.before + blockIdx.x * g.pitch;
    uint32_t before = 0;
    for (int64_t b0 = 0; b0 < workgroups; b0 += 256) {
        const int64_t b = b0 + threadIdx.x;
        const uint32_t n = b < workgroups ? counts[b] : 0;
        const uint32_t incl = wave_prefix(n);
        if (lane_id() == kWave - 1) part[w] = incl;
        __syncthreads();
        uint32_t add = before, all = 0;
        for (int i = 0; i < 4; ++i) {
            if (i < w) add += part[i];
            all += part[i];
        }
        if (b < workgroups) out[b] = add + incl - n;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) g.sizes[blockIdx.x] = (int32_t)before;
}

// The workgroups of the choice again: their pairs' places.
__global__ __launch_bounds__(256) void route_place_kernel(RouteArgs g, int64_t workgroups) {
    __shared__ uint64_t mask[kRouteExperts];
    __shared__ uint32_t first[kRouteExperts], before[kRouteExperts], part[4];
    const int64_t row0 = (int64_t)blockIdx.x * kRouteRows;
    for (int e = threadIdx.x; e < g.E; e += 256) {
        mask[e] = 0;
        if (workgroups > kDirect) {
            first[e] = g.sizes[e];
            before[e] = g.before[e * g.pitch + blockIdx.x];
        } else {
            const uint32_t *counts = reinterpret_cast<const uint32_t *>(g.counts + e * g.pitch);
            uint32_t sum = 0, all = 0;
            for (int i = 0; i < workgroups; i += 4) {  // sums of 4 bytes, those before this workgroup and all
                const uint32_t c = counts[i / 4];
                const int here = (int)blockIdx.x - i, there = (int)workgroups - i;
                sum = __builtin_amdgcn_sad_u8(here >= 4 ? c : here <= 0 ? 0 : c & (0xffffffffu >> (32 - 8 * here)), 0, sum);
                all = __builtin_amdgcn_sad_u8(there >= 4 ? c : c & (0xffffffffu >> (32 - 8 * there)), 0, all);
            }
            first[e] = all;
            before[e] = sum;
            if (blockIdx.x == 0) g.sizes[e] = (int32_t)all;
        }
    }
    __syncthreads();
    const int64_t rows = g.T - row0 < kRouteRows ? g.T - row0 : kRouteRows;
    const int32_t *chosen = g.experts + row0 * g.k;
    for (int i = threadIdx.x; i < rows * g.k; i += 256) {
        const int32_t e = chosen[i];
        if (e >= 0) set_bit(&mask[e], i / g.k);
    }
    const uint32_t total = prefix_experts<256>(first, g.E, part);
    for (int e = threadIdx.x; e < g.E; e += 256) first[e] += before[e];
    __syncthreads();
    place_pairs<256>(g, row0, mask, first, chosen, total);
}

struct RouteGradArgs {
    const float *g, *weights;
    const void *logits;
    const int32_t *experts;
    void *d;
    int64_t T, ld;
    int E, k, normalize;
};

// d logits: w_j (g_j - sum_c w_c g_c) where an expert was chosen, and, with a softmax over all, -p_e sum_c w_c g_c elsewhere.
// 16 lanes a row; the row is put together in LDS and written 16 bytes a lane.
template <typename T, int V>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteGradArgs a) {
    constexpr int ROW = 16 * V;
    __shared__ __attribute__((aligned(16))) T out[16][ROW];
    const int lane = threadIdx.x & 15, r = threadIdx.x / 16;
    const int64_t t = (int64_t)blockIdx.x * 16 + r;
    const bool there = t < a.T;
    float w = 0.0f, g = 0.0f;
    int32_t expert = -1;
    if (there && lane < a.k) {
        w = a.weights[t * a.k + lane];
        g = a.g[t * a.k + lane];
        expert = a.experts[t * a.k + lane];
        if (expert >= a.E) expert = -1;  // not of this router: no gradient
    }
    const float inner = row_sum(expert >= 0 ? w * g : 0.0f);
    if (a.normalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[r][lane * V + i] = T(0.0f);
    } else {
        float x[V];
        if (there) load_logits(static_cast<const T *>(a.logits) + t * a.ld, lane, a.E, x);
        else
            for (int i = 0; i < V; ++i) x[i] = -__builtin_inff();
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t key = order_key(x[i]);
            best = key > best ? key : best;
        }
        const float top = key_value(row_max(best));  // of a row of -inf: not used
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            x[i] = x[i] == -__builtin_inff() ? 0.0f : expf(x[i] - top);
            s += x[i];
        }
        s = row_sum(s);
#pragma unroll
        for (int i = 0; i < V; ++i) out[r][lane * V + i] = T(x[i] == 0.0f ? 0.0f : -(x[i] / s) * inner);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");  // a row's 16 lanes are in one wavefront
    __builtin_amdgcn_wave_barrier();
    if (expert >= 0) out[r][expert] = T(w * (g - inner));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    if (!there) return;
    T *d = static_cast<T *>(a.d) + t * a.E;
    constexpr int C = 16 / sizeof(T);
    const bool whole = ((reinterpret_cast<uintptr_t>(a.d) | (uint64_t)(a.E * sizeof(T))) & 15) == 0;
    if (whole) {
        for (int c = lane * C; c < a.E; c += 16 * C) *reinterpret_cast<uintx4 *>(d + c) = *reinterpret_cast<const uintx4 *>(&out[r][c]);
    } else {
        for (int c = lane; c < a.E; c += 16) d[c] = out[r][c];
    }
}

template <typename T, int V>
void launch_choose(const RouteArgs &g, int64_t workgroups, hipStream_t s) {
    if (workgroups == 1) hipLaunchKernelGGL((route_choose_kernel<T, V, true>), dim3(1), dim3(kChooseThreads<V>), 0, s, g);
    else hipLaunchKernelGGL((route_choose_kernel<T, V, false>), dim3((unsigned)workgroups), dim3(kChooseThreads<V>), 0, s, g);
}

template <typename T>
void launch_choose(const RouteArgs &g, int64_t workgroups, hipStream_t s) {
    if (g.E <= 64) launch_choose<T, 4>(g, workgroups, s);
    else if (g.E <= 128) launch_choose<T, 8>(g, workgroups, s);
    else if (g.E <= 256) launch_choose<T, 16>(g, workgroups, s);
    else if (g.E <= 512) launch_choose<T, 32>(g, workgroups, s);
    else launch_choose<T, 64>(g, workgroups, s);
}

template <typename T>
void launch_route_grad(const RouteGradArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(a.T, 16)), block(256);
    if (a.E <= 64) hipLaunchKernelGGL((route_grad_kernel<T, 4>), grid, block, 0, s, a);
    else if (a.E <= 128) hipLaunchKernelGGL((route_grad_kernel<T, 8>), grid, block, 0, s, a);
    else if (a.E <= 256) hipLaunchKernelGGL((route_grad_kernel<T, 16>), grid, block, 0, s, a);
    else if (a.E <= 512) hipLaunchKernelGGL((route_grad_kernel<T, 32>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((route_grad_kernel<T, 64>), grid, block, 0, s, a);
}

inline int64_t route_workgroups(int64_t T) { return ceil_div(T, kRouteRows); }
inline int64_t route_pitch(int64_t workgroups) { return ceil_div(workgroups, 64) * 64; }

}  // namespace trt

using namespace trt;

extern "C" size_t trt_route_workspace_bytes(int64_t T, int64_t E) {
    if (T <= kRouteRows || E <= 0 || T >= (int64_t)1 << 31) return 0;
    const int64_t n = route_workgroups(T), pitch = route_pitch(n);
    return (size_t)(E * pitch * (n > kDirect ? 5 : 1));
}

extern "C" int trt_route(const void *logits, float *weights, int32_t *experts, int32_t *rows, int32_t *slots, int32_t *sizes, int64_t T,
                         int64_t E, int64_t k, int64_t ld, int dtype, int normalize, void *workspace, size_t workspace_bytes,
                         void *stream) {
    if (!logits || !weights || !experts || !rows || !slots || !sizes || T <= 0 || E <= 0 || k <= 0 || k > E) return TRT_E_INVALID;
    if (dtype != TRT_F32 && dtype != TRT_F16 && dtype != TRT_BF16) return TRT_E_INVALID;
    if (ld < 0) return TRT_E_LAYOUT;
    if (E > kRouteExperts || k > kRouteMost || T * k >= (int64_t)1 << 31 || T >= (int64_t)1 << 31) return TRT_E_RANGE;
    const size_t need = trt_route_workspace_bytes(T, E);
    if (need && (!workspace || workspace_bytes < need)) return TRT_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return TRT_E_LAYOUT;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t n = route_workgroups(T);
    RouteArgs g = {};
    g.logits = logits, g.weights = weights, g.experts = experts, g.rows = rows, g.slots = slots, g.sizes = sizes;
    g.T = T, g.ld = ld, g.pitch = route_pitch(n), g.E = (int)E, g.k = (int)k, g.normalize = normalize;
    g.before = static_cast<uint32_t *>(workspace);
    g.counts = static_cast<uint8_t *>(workspace) + (n > kDirect ? 4 * E * g.pitch : 0);
    switch (dtype) {
        case TRT_F32: launch_choose<float>(g, n, s); break;
        case TRT_F16: launch_choose<_Float16>(g, n, s); break;
        default: launch_choose<__bf16>(g, n, s); break;
    }
    if (n > kDirect) hipLaunchKernelGGL(route_prefix_kernel, dim3((unsigned)E), dim3(256), 0, s, g, n);
    if (n > 1) hipLaunchKernelGGL(route_place_kernel, dim3((unsigned)n), dim3(256), 0, s, g, n);
    return (int)hipGetLastError();
}

extern "C" int trt_route_grad(const float *g, const void *logits, const float *weights, const int32_t *experts, void *d, int64_t T,
                              int64_t E, int64_t k, int64_t ld, int dtype, int normalize, void *stream) {
    if (!g || !logits || !weights || !experts || !d || T <= 0 || E <= 0 || k <= 0 || k > E) return TRT_E_INVALID;
    if (ld < 0) return TRT_E_LAYOUT;
    if (E > kRouteExperts || k > kRouteMost || T * k >= (int64_t)1 << 31 || T >= (int64_t)1 << 31) return TRT_E_RANGE;
    RouteGradArgs a = {g, weights, logits, experts, d, T, ld, (int)E, (int)k, normalize};
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TRT_F32: launch_route_grad<float>(a, s); break;
        case TRT_F16: launch_route_grad<_Float16>(a, s); break;
        case TRT_BF16: launch_route_grad<__bf16>(a, s); break;
        default: return TRT_E_INVALID;
    }
    return (int)hipGetLastError();
}
