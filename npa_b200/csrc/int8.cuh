// Rows and weights in 8-bit integers with one scale per row: what the kernels of int8.cu share.
//
//     scale = max(fl32(max |x| / most), 2^-126),   code = x / scale rounded to nearest, ties to even,   most = 127, or 255 unsigned
//
// The code is that of the exact quotient: the scale is the only rounding in front of it, so that every evaluation of the definition,
// in 32 or 64 bits, finds the same codes.  The floor keeps the scale a normal number, and rows of zeros away from 0 / 0.  A row that
// holds an infinity or a NaN has the scale NaN and codes of zero: everything computed from it is NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace npa {

constexpr float kScaleFloor = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Magnitudes are compared as integers: a NaN is above infinity, which is above every number.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// What is quantised of a value: unsigned codes have none for numbers below zero (an infinity of either sign is seen all the same).
template <bool UNSIGNED>
__device__ __forceinline__ float quantizable(float v) { return UNSIGNED && v < 0.f && magnitude(v) < 0x7f800000u ? 0.f : v; }

// Scale of a row from its largest magnitude; `inverse` is near 1 / scale.
__device__ __forceinline__ float row_scale(unsigned largest, float most, float &inverse) {
    if (largest >= 0x7f800000u) {
        inverse = 0.f;
        return __int_as_float(0x7fc00000);
    }
    const float s = fmaxf(__fdiv_rn(__uint_as_float(largest), most), kScaleFloor);
    inverse = __frcp_rn(s);
    return s;
}

// x / scale rounded to nearest, ties to even.  x * inverse is within 2^-22 of the quotient, relatively, so the first guess is right or
// off by one next to a border; the remainder x - r scale is exact (a multiple of the smaller unit of the two, below the scale), and
// says which.
__device__ __forceinline__ int row_code(float x, float scale, float inverse) {
    if (inverse == 0.f) return 0;
    float r = rintf(x * inverse);
    const float rest = __fmaf_rn(-r, scale, x), half = 0.5f * scale, off = fabsf(rest);
    if (off > half || (off == half && ((int)r & 1))) r += copysignf(1.f, rest);
    return (int)r;
}

__device__ __forceinline__ unsigned warp_max(unsigned v) { return __reduce_max_sync(kFull, v); }

}  // namespace npa
