// Activations in 8 bits, as a checkpoint for the backward pass holds them.
//
// Groups of 32 columns of a row share a power of two:  value = code * 2^(E - 133),  |code| <= 127,  E one byte per group, where
//
//     E = ((bits(max |x|) + 0x10000) >> 23), between 7 and 254
//
// is the smallest exponent in whose units the largest value rounds to at most 127 (the largest is 64 to 127.5 units: rounding in its
// own binade never reaches 128 below 0x7f0000 of the fraction).  A power of two costs up to a bit against max / 127, and buys that
// both ways are exact but for the one rounding to the code, and that a value held so is a number of 8 significant bits: products with
// it need no tail on the tensor cores.  A group that holds an infinity or a NaN has E = 255 and all its values are NaN.
#pragma once
#include "int8.cuh"

namespace npa {

constexpr int kRowsGroup = 32;

__host__ __device__ inline int rows8_groups(int cols) { return (cols + kRowsGroup - 1) / kRowsGroup; }
__host__ __device__ inline long long rows8_pitch(int cols) { return (cols + 15) / 16 * 16; }

__device__ __forceinline__ unsigned rows8_exponent(unsigned largest) {
    return largest >= 0x7f800000u ? 255u : min(max((largest + 0x10000u) >> 23, 7u), 254u);
}
// 2^(133 - E): times it, a value is in units of its group (E = 255: zero, so that codes are zero).
__device__ __forceinline__ float rows8_to_units(unsigned e) { return e == 255u ? 0.f : __uint_as_float((133u + 127u - e) << 23); }
// 2^(E - 133), or NaN.
__device__ __forceinline__ float rows8_unit(unsigned e) { return e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((e - 133u + 127u) << 23); }
__device__ __forceinline__ int rows8_code(float x, float to_units) {
    return to_units == 0.f ? 0 : max(-127, min(127, __float2int_rn(x * to_units)));
}
// Codes of N values of a group, in their lowest bytes: rounded by adding 1.5 * 2^23.  Only the last binade (up to 128 units) and groups
// that are not finite need rows8_code.
template <int N>
__device__ __forceinline__ void rows8_codes(const float (&x)[N], unsigned e, float to_units, unsigned (&code)[N]) {
#pragma unroll
    for (int q = 0; q < N; ++q) code[q] = __float_as_uint(__fmaf_rn(x[q], to_units, kRoundWhole));
    if (e >= 254u) {
#pragma unroll
        for (int q = 0; q < N; ++q) code[q] = (unsigned)rows8_code(x[q], to_units);
    }
}
// Four codes as numbers: each byte, 128 added, becomes the last of 2^23's.
__device__ __forceinline__ void rows8_numbers(unsigned codes, float (&v)[4]) {
    const unsigned u = codes ^ 0x80808080u;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + q)) - 8388736.f;
}

// mlp_checkpoint.cu: the sizes that the MLP with a checkpoint takes.
int check_mlp8(const char *me, int64_t rows, int32_t in_dim, int32_t out_dim);

}  // namespace npa
