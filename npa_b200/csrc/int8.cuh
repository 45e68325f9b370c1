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

#include <type_traits>

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

// Codes of N values: x * inverse rounded to a whole number by adding 1.5 * 2^23, whose lowest byte is the code.  It is within 3e-5 of the
// quotient (255 * 2^-23), so it is the right one unless that lies so near a border; the largest remainder says whether there is such
// a value among them, or one half way between two codes: then row_code looks at each (`true`, one value in 10^5).
constexpr float kRoundWhole = 12582912.f;
template <int N>
__device__ __forceinline__ bool quick_codes(const float (&x)[N], float scale, float inverse, unsigned (&code)[N]) {
    float rest = 0.f;
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const float f = __fmaf_rn(x[q], inverse, kRoundWhole);
        code[q] = __float_as_uint(f);
        rest = fmaxf(rest, fabsf(__fmaf_rn(kRoundWhole - f, scale, x[q])));
    }
    return rest >= 0.5f * scale;
}
static __device__ __noinline__ unsigned row_code_out_of_line(float x, float scale, float inverse) { return (unsigned)row_code(x, scale, inverse); }
// (FAR: where many copies of this would crowd the instructions that run; replayed graphs of mlp_int8 11.4 us for 2,500 rows instead of 12.3, 80.6 for
// 262,144 instead of 84.0.)
template <int N, bool FAR = false>
__device__ __forceinline__ void row_codes(const float (&x)[N], float scale, float inverse, unsigned (&code)[N]) {
    if (quick_codes(x, scale, inverse, code)) {
#pragma unroll
        for (int q = 0; q < N; ++q) code[q] = FAR ? row_code_out_of_line(x[q], scale, inverse) : (unsigned)row_code(x[q], scale, inverse);
    }
}
// The lowest bytes of four codes.
__device__ __forceinline__ unsigned pack_codes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <int LANES = 32>
__device__ __forceinline__ unsigned warp_max(unsigned v) {
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) v = max(v, __shfl_xor_sync(kFull, v, d));
    return v;
}
// The larger magnitude; NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return max(a, b); }
// Eight maxima over the lanes of a group of LANES at once: the lanes share the values out while they halve, 8 or 9 shuffles instead of
// 32 or 40.  That of value r comes to lanes r LANES / 8 and up of the group.
template <int LANES = 32, typename V>
__device__ __forceinline__ V gather_max8(V (&v)[8]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 4, d = LANES / 2; n >= 1; n /= 2, d /= 2) {
        const bool up = lane & d;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const V keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
            v[i] = larger(keep, __shfl_xor_sync(kFull, send, d));
        }
    }
    V m = v[0];
#pragma unroll
    for (int d = LANES / 16; d >= 1; d /= 2) m = larger(m, __shfl_xor_sync(kFull, m, d));
    return m;
}
template <int LANES = 32>
__device__ __forceinline__ int max8_lane(int r) { return (threadIdx.x & 31 & ~(LANES - 1)) + r * (LANES / 8); }
// And each to all lanes of its group.
template <int LANES = 32>
__device__ __forceinline__ void warp_max8(unsigned (&v)[8]) {
    const unsigned m = gather_max8<LANES>(v);
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = __shfl_sync(kFull, m, max8_lane<LANES>(r));
}

// V values at p, of which `left` exist; in loads of W bytes.
template <typename T, int V, int W = 16>
struct Values {
    using Word = std::conditional_t<W == 16, uint4, uint2>;
    union {
        Word word[V == 1 ? 1 : V * (int)sizeof(T) / W];
        T value[V];
    };
    __device__ __forceinline__ void load(const T *__restrict__ p, int left) {
        if constexpr (V > 1) {
            if (left >= V) {
#pragma unroll
                for (int q = 0; q < V * (int)sizeof(T) / W; ++q) word[q] = __ldg(reinterpret_cast<const Word *>(p) + q);
                return;
            }
        }
#pragma unroll
        for (int q = 0; q < V; ++q) value[q] = q < left ? p[q] : from_float<T>(0.f);
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = as_float(value[q]);
    }
    __device__ __forceinline__ Values() {}
    __device__ __forceinline__ Values &operator=(const Values &from) {
#pragma unroll
        for (int q = 0; q < (int)(sizeof(word) / sizeof(Word)); ++q) word[q] = from.word[q];
        return *this;
    }
};
template <typename T, int V, int W = 16>
__device__ __forceinline__ void load_values(const T *__restrict__ p, int left, float (&v)[V]) {
    Values<T, V, W> r;
    r.load(p, left);
    r.get(v);
}
// V codes to p, of which `left` exist; `aligned`: p is a multiple of V.
template <int V>
__device__ __forceinline__ void store_codes(uint8_t *p, int left, bool aligned, const unsigned (&code)[V]) {
    if constexpr (V == 8) {
        if (left >= V && aligned) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(pack_codes(code[0], code[1], code[2], code[3]), pack_codes(code[4], code[5], code[6], code[7]));
            return;
        }
    }
    {
#pragma unroll
        for (int q = 0; q < V; ++q)
            if (q < left) p[q] = (uint8_t)code[q];
    }
}

// ---- rows put together in shared memory ----------------------------------------------------------------------------------
// 16 values (`left` of them exist) of a row in a tile whose rows follow one another without a gap, lane = row.  Word by word the lanes meet
// in a bank as often as 32 and the length have a factor in common (32 ways for 32, 64, 96, 128, 160 columns); rows of a multiple of four
// columns go by 16 bytes, each lane beginning with another of its four pieces where rows start in the same banks, which leaves two ways at most.
__device__ __forceinline__ int first_piece(int cols, int lane) {
    const int common = min((cols / 4) & -(cols / 4), 8);
    return ((lane & 7) * common >> 3) & 3;
}
__device__ __forceinline__ void put_16_pieces(float *to, int left, int first, float (&v)[16]) {
    float w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = first & 1 ? v[(j + 4) % 16] : v[j];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = first & 2 ? w[(j + 8) % 16] : w[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = 4 * ((i + first) & 3);
        if (k < left) *reinterpret_cast<float4 *>(to + k) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
}
__device__ __forceinline__ void put_16(float *to, int left, int cols, int lane, float (&v)[16]) {
    if (cols % 4 == 0) {
        put_16_pieces(to, left, first_piece(cols, lane), v);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < left) to[j] = v[j];
    }
}

// ---- the product -----------------------------------------------------------------------------------------------------
struct Int8Args {
    const void *x;       // [rows, in] codes, or values that the kernel for few rows quantises
    const int8_t *w;     // [out, in], rows 16-byte aligned
    long long x_pitch, w_pitch;  // in elements
    int x_type;
    const float *x_scales, *w_scales;
    const int *w_sums;   // rows of codes that were shifted from unsigned to signed by 128: sums of the channels' weights, else NULL
    const void *bias;    // [out] or NULL
    int bias_type, relu, out_type;
    void *out;           // [rows, out]
    long long rows;
    int in, out_dim;
};

__device__ __forceinline__ float load_value(const void *p, int type, long long at) {
    if (type == NPA_FLOAT32) return static_cast<const float *>(p)[at];
    if (type == NPA_FLOAT16) return __half2float(static_cast<const __half *>(p)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
}
// No product is contracted with the sum behind it: the roundings are those of the definition.
__device__ __forceinline__ float int8_value(int sum, float s, float t, bool has_bias, float bias, bool relu) {
    float v = __fmul_rn(__int2float_rn(sum), __fmul_rn(s, t));
    if (has_bias) v = __fadd_rn(v, bias);
    return relu && v < 0.f ? 0.f : v;  // (a NaN stays one)
}

// int8_tcgen05.cu: the product of codes on the tensor cores; x and w 16-byte aligned with pitches of multiples of 16, x signed.
int launch_int8_tcgen05(const char *me, const Int8Args &a, cudaStream_t st);

// int8_mlp.cu: both layers in one kernel, where the arrays lie as it wants them.
bool mlp_int8_fused(const float *z, long long z_pitch, const void *w1, long long w1_pitch, const void *w2, long long w2_pitch, long long rows, int in, int hidden,
                    int out);
int launch_mlp_int8(const char *me, const float *z, const void *w1, long long w1_pitch, const float *t1, const float *b1, const void *w2, long long w2_pitch,
                    const float *t2, float *y, long long rows, int in, int out, cudaStream_t st);

}  // namespace npa
