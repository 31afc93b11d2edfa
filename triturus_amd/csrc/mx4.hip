// The microscaled 4-bit format: quantisation of rows and back.
//
// Blocks of 32 values along a row share a power of two (OCP Microscaling Formats v1.0, MXFP4): with
// e = floor(log2 max |x|) - 2, held as a byte e + 127, every value is x / 2^e rounded to the nearest of
// 0, 1/2, 1, 3/2, 2, 3, 4, 6 (E2M1: ties to the even code, beyond 6 to 6) with its sign.  A block that holds a NaN or an
// infinity has scale 255, which stands for NaN.  A block is 16 bytes of codes (the even value in the low
// half of a byte) and one byte of scale; a row's last block is filled up with zeros.
//
// Bound: HBM.  A lane takes 16 bytes of the row (32 of fp32), so 4 lanes make a block; the largest is found in 2
// lane steps and the codes by the conversion instructions, 2 values each.  16384 x 4096 of bf16: 33 us to codes (5.2 TB/s read
// and written), 38 us back (4.5 TB/s).
#include "mx4.hpp"

namespace trt {

constexpr int kPart = 8;                // values of a lane
constexpr int kParts = 32 / kPart;      // lanes of a block

// x: rows of K values, row stride ld; codes: rows of 16 * blocks bytes, scales: rows of `blocks` bytes, both dense.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T *__restrict__ x, uint32_t *__restrict__ codes,
                                                           uint8_t *__restrict__ scales, uint32_t parts, int64_t K, int64_t ld,
                                                           Divider per_row) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= parts) return;  // blocks end with a group of four lanes
    const uint32_t row = divide(i, per_row), at = i - row * per_row.d;
    T v[kPart];
    load_values(x + row * ld + at * kPart, K - (int64_t)at * kPart, v);
    uint32_t top = top_bits(v);
    top = max_u(top, __builtin_amdgcn_mov_dpp(top, 0xB1, 0xf, 0xf, true));  // lanes 1 0 3 2 of each four
    top = max_u(top, __builtin_amdgcn_mov_dpp(top, 0x4E, 0xf, 0xf, true));  // lanes 2 3 0 1
    const uint32_t scale = block_scale(top);
    uint32_t word[1];
    codes_of(v, scale, word);
    codes[i] = word[0];
    if (i % kParts == 0) scales[i / kParts] = (uint8_t)scale;
}

// y: dense rows of K values; codes and scales with row strides in bytes.
template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                             T *__restrict__ y, uint32_t parts, int64_t K, int64_t ld_codes,
                                                             int64_t ld_scales, Divider per_row, bool whole) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= parts) return;
    const uint32_t row = divide(i, per_row), at = i - row * per_row.d;
    uint32_t code;
    __builtin_memcpy(&code, codes + row * ld_codes + at * 4, 4);
    const uint32_t scale = scales[row * ld_scales + at / kParts];
    // 2^(scale - 127) as two factors, both normal numbers
    const float a = __builtin_bit_cast(float, ((scale >> 1) + 64) << 23), b = __builtin_bit_cast(float, (scale - (scale >> 1) + 63) << 23);
    struct alignas(16) { T v[kPart]; } out;
#pragma unroll
    for (int u = 0; u < kPart; ++u) {
        const uint32_t c = code >> (4 * u);
        // E2M1 as the top bits of a float: exponents 1..3 become 127..129 by a multiplication that also scales subnormals
        const float m = __builtin_bit_cast(float, (c & 7) << 22) * 0x1p126f;
        const float f = scale == 255 ? __builtin_nanf("") : (m * a) * b;
        out.v[u] = (T)((c & 8) ? -f : f);
    }
    const int64_t left = K - (int64_t)at * kPart;
    T *p = y + row * K + at * kPart;
    if (whole) {
        *reinterpret_cast<decltype(out) *>(p) = out;
    } else {
#pragma unroll
        for (int u = 0; u < kPart; ++u)
            if (u < left) p[u] = out.v[u];
    }
}

constexpr int64_t kMostParts = (int64_t)1 << 30;  // of one launch: a lane's number has 31 bits

template <typename T>
int launch_quantize(const T *x, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t K, int64_t ld, hipStream_t s) {
    const int64_t blocks = ceil_div(K, 32), per = blocks * kParts;
    for (int64_t r = 0; r < rows;) {
        const int64_t n = rows - r < kMostParts / per ? rows - r : kMostParts / per;
        const uint32_t parts = (uint32_t)(n * per);
        hipLaunchKernelGGL(mx4_quantize_kernel<T>, dim3((unsigned)ceil_div(parts, 256)), dim3(256), 0, s, x + r * ld,
                           reinterpret_cast<uint32_t *>(codes + r * blocks * 16), scales + r * blocks, parts, K, ld, divider((uint32_t)per));
        r += n;
    }
    return (int)hipGetLastError();
}

template <typename T>
int launch_dequantize(const uint8_t *codes, const uint8_t *scales, T *y, int64_t rows, int64_t K, int64_t ld_codes, int64_t ld_scales,
                      hipStream_t s) {
    const int64_t per = ceil_div(K, kPart);
    const bool whole = K % kPart == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
    for (int64_t r = 0; r < rows;) {
        const int64_t n = rows - r < kMostParts / per ? rows - r : kMostParts / per;
        const uint32_t parts = (uint32_t)(n * per);
        hipLaunchKernelGGL(mx4_dequantize_kernel<T>, dim3((unsigned)ceil_div(parts, 256)), dim3(256), 0, s, codes + r * ld_codes,
                           scales + r * ld_scales, y + r * K, parts, K, ld_codes, ld_scales, divider((uint32_t)per), whole);
        r += n;
    }
    return (int)hipGetLastError();
}

}  // namespace trt

using namespace trt;

extern "C" int trt_mx4_quantize(const void *x, void *codes, void *scales, int64_t rows, int64_t K, int64_t ldx, int dtype, void *stream) {
    if (!x || !codes || !scales || rows <= 0 || K <= 0) return TRT_E_INVALID;
    if (ldx < 0 || (reinterpret_cast<uintptr_t>(codes) & 3)) return TRT_E_LAYOUT;
    if (K > (int64_t)1 << 30) return TRT_E_RANGE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint8_t *c = static_cast<uint8_t *>(codes), *e = static_cast<uint8_t *>(scales);
    switch (dtype) {
        case TRT_F32: return launch_quantize(static_cast<const float *>(x), c, e, rows, K, ldx, s);
        case TRT_F16: return launch_quantize(static_cast<const _Float16 *>(x), c, e, rows, K, ldx, s);
        case TRT_BF16: return launch_quantize(static_cast<const __bf16 *>(x), c, e, rows, K, ldx, s);
        default: return TRT_E_INVALID;
    }
}

extern "C" int trt_mx4_dequantize(const void *codes, const void *scales, void *y, int64_t rows, int64_t K, int64_t ld_codes,
                                  int64_t ld_scales, int dtype, void *stream) {
    if (!codes || !scales || !y || rows <= 0 || K <= 0) return TRT_E_INVALID;
    if (ld_codes < 0 || ld_scales < 0) return TRT_E_LAYOUT;
    if (K > (int64_t)1 << 30) return TRT_E_RANGE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint8_t *c = static_cast<const uint8_t *>(codes), *e = static_cast<const uint8_t *>(scales);
    switch (dtype) {
        case TRT_F32: return launch_dequantize(c, e, static_cast<float *>(y), rows, K, ld_codes, ld_scales, s);
        case TRT_F16: return launch_dequantize(c, e, static_cast<_Float16 *>(y), rows, K, ld_codes, ld_scales, s);
        case TRT_BF16: return launch_dequantize(c, e, static_cast<__bf16 *>(y), rows, K, ld_codes, ld_scales, s);
        default: return TRT_E_INVALID;
    }
}
