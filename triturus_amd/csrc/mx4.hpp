// Quantisation of blocks of 32 values to the microscaled 4-bit format.
#pragma once

#include "grouped.hpp"

namespace trt {

__device__ __forceinline__ uint32_t max_u(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The largest magnitude of N values, as the bits of a float: infinities and NaN are above all numbers.
template <typename T, int N>
__device__ __forceinline__ uint32_t top_bits(const T (&v)[N]) {
    if constexpr (sizeof(T) == 2) {  // two at a time
        typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
        ushort2v top = {0, 0};
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint32_t u;
            __builtin_memcpy(&u, &v[i], 4);
            top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2v, u & 0x7fff7fffu));
        }
        const unsigned short one = top[0] > top[1] ? top[0] : top[1];
        return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(T, one));
    } else {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) top = max_u(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
        return top;
    }
}

// The biased exponent that a block with this largest magnitude is stored under.
__device__ __forceinline__ uint32_t block_scale(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

template <typename T, int SEL>
__device__ __forceinline__ uint32_t code_pair(uint32_t codes, const T *v, float by) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], by, SEL);
    } else {
        typedef T pair __attribute__((ext_vector_type(2)));
        const pair p = {v[0], v[1]};
        if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, p, by, SEL);
        else return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, p, by, SEL);
    }
}

// 8 codes a word under a block's scale.  The conversion divides by a power of two that has to be a normal number, and takes no
// subnormal values: blocks whose largest magnitude is below 2^-93 (never fp16's) are moved up by 2^32 before, exactly.
template <typename T, int N>
__device__ __forceinline__ void codes_of(const T (&v)[N], uint32_t scale, uint32_t (&codes)[N / 8]) {
#pragma unroll
    for (int w = 0; w < N / 8; ++w) codes[w] = 0;
    if (scale == 255) return;
    if (scale >= 32 || __is_same(T, _Float16)) {
        const float by = __builtin_bit_cast(float, (scale ? scale : 127) << 23);  // 0: all values are 0
#pragma unroll
        for (int w = 0; w < N / 8; ++w) {
            codes[w] = code_pair<T, 0>(codes[w], v + 8 * w, by);
            codes[w] = code_pair<T, 1>(codes[w], v + 8 * w + 2, by);
            codes[w] = code_pair<T, 2>(codes[w], v + 8 * w + 4, by);
            codes[w] = code_pair<T, 3>(codes[w], v + 8 * w + 6, by);
        }
    } else {
        const float by = __builtin_bit_cast(float, (scale + 32) << 23);
#pragma unroll
        for (int w = 0; w < N / 8; ++w) {
            float u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = (float)v[8 * w + i] * 0x1p32f;
            codes[w] = code_pair<float, 0>(codes[w], u, by);
            codes[w] = code_pair<float, 1>(codes[w], u + 2, by);
            codes[w] = code_pair<float, 2>(codes[w], u + 4, by);
            codes[w] = code_pair<float, 3>(codes[w], u + 6, by);
        }
    }
}

// N values from p on, of which `left` exist (<= 0: none); the others are 0.
template <typename T, int N>
__device__ __forceinline__ void load_values(const T *p, int64_t left, T (&v)[N]) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < N / V; ++i) {
        const uintx4 u = load_chunk(p + i * V, left - i * V);
        __builtin_memcpy(&v[i * V], &u, 16);
    }
}

}  // namespace trt
