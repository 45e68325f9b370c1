// Products in 8-bit integers: rows quantised with a scale each, weights with a scale for each output channel.
//
//     out[m, n] = act( float(sum_k q[m, k] w[n, k]) * (s[m] * t[n]) + bias[n] )
//
// The sum is one of integers and exact (a chain of 65,536 products of 255 and 127 stays below 2^31); behind it are three roundings of
// 32 bits -- the product of the scales, its product with the sum, the bias -- and the one to the type of the output.
#include "int8.cuh"

namespace npa {

constexpr int kInt8MaxIn = 65536;

// ---- rows into codes -------------------------------------------------------------------------------------------------
// A warp per row: the largest magnitude, then the codes, four to a store.  Reading and writing memory is all there is to it.
template <typename T, bool UNSIGNED>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T *__restrict__ x, long long pitch, long long rows, int cols,
                                                            uint8_t *__restrict__ codes, long long codes_pitch, float *__restrict__ scales) {
    after_previous_kernel();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const T *p = x + row * pitch;
    unsigned largest = 0;
    for (int k = lane; k < cols; k += 32) largest = max(largest, magnitude(quantizable<UNSIGNED>(as_float(p[k]))));
    float inverse;
    const float scale = row_scale(warp_max(largest), UNSIGNED ? 255.f : 127.f, inverse);
    for (int k = lane; k < cols; k += 32) codes[row * codes_pitch + k] = (uint8_t)row_code(quantizable<UNSIGNED>(as_float(p[k])), scale, inverse);
    if (lane == 0) scales[row] = scale;
}

template <typename T, typename Code>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const Code *__restrict__ codes, long long codes_pitch, const float *__restrict__ scales,
                                                              long long rows, int cols, T *__restrict__ out) {
    after_previous_kernel();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const float scale = scales[row];
    for (int k = lane; k < cols; k += 32) out[row * cols + k] = from_float<T>((float)codes[row * codes_pitch + k] * scale);
}

// ---- the product -----------------------------------------------------------------------------------------------------
struct Int8Args {
    const uint8_t *x;   // [rows, in] codes, signed or not
    const int8_t *w;    // [out, in]
    long long x_pitch, w_pitch;
    const float *x_scales, *w_scales;
    const void *bias;   // [out] or NULL
    int bias_type, relu, x_unsigned;
    void *out;          // [rows, out]
    long long rows;
    int in, out_dim;
};

__device__ __forceinline__ float load_bias(const void *bias, int type, int n) {
    if (!bias) return 0.f;
    if (type == NPA_FLOAT32) return static_cast<const float *>(bias)[n];
    if (type == NPA_FLOAT16) return __half2float(static_cast<const __half *>(bias)[n]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(bias)[n]);
}
// No product is contracted with the sum behind it: the roundings are those of the definition.
__device__ __forceinline__ float int8_value(int sum, float s, float t, bool has_bias, float bias, bool relu) {
    float v = __fmul_rn(__int2float_rn(sum), __fmul_rn(s, t));
    if (has_bias) v = __fadd_rn(v, bias);
    return relu && v < 0.f ? 0.f : v;  // (a NaN stays one)
}

constexpr int kTileM = 32, kTileN = 64, kTileK = 64;

template <typename T>
__global__ void __launch_bounds__(256) int8_tile_kernel(const __grid_constant__ Int8Args a) {
    after_previous_kernel();
    __shared__ int xs[kTileM][kTileK / 4 + 1], ws[kTileN][kTileK / 4 + 1];
    const long long row0 = (long long)blockIdx.x * kTileM;
    const int n0 = blockIdx.y * kTileN, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // columns tx, tx + 32; rows ty, ty + 8, ...
    int acc[4][2] = {};
    for (int k0 = 0; k0 < a.in; k0 += kTileK) {
        for (int q = threadIdx.x; q < (kTileM + kTileN) * kTileK; q += 256) {
            const int r = q / kTileK, k = q % kTileK;
            uint8_t v = 0;
            if (r < kTileM) {
                if (row0 + r < a.rows && k0 + k < a.in) v = a.x[(row0 + r) * a.x_pitch + k0 + k];
                reinterpret_cast<uint8_t *>(xs[r])[k] = v;
            } else {
                if (n0 + r - kTileM < a.out_dim && k0 + k < a.in) v = (uint8_t)a.w[(long long)(n0 + r - kTileM) * a.w_pitch + k0 + k];
                reinterpret_cast<uint8_t *>(ws[r - kTileM])[k] = v;
            }
        }
        __syncthreads();
        for (int k = 0; k < kTileK / 4; ++k)
            for (int j = 0; j < 2; ++j)
                for (int i = 0; i < 4; ++i) {
                    const int wv = ws[tx + 32 * j][k], xv = xs[ty + 8 * i][k];
                    if (a.x_unsigned) asm("dp4a.u32.s32 %0, %1, %2, %0;" : "+r"(acc[i][j]) : "r"(xv), "r"(wv));
                    else acc[i][j] = __dp4a(xv, wv, acc[i][j]);
                }
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 2; ++j) {
            const long long row = row0 + ty + 8 * i;
            const int n = n0 + tx + 32 * j;
            if (row < a.rows && n < a.out_dim)
                static_cast<T *>(a.out)[row * a.out_dim + n] = from_float<T>(int8_value(
                    acc[i][j], a.x_scales[row], a.w_scales[n], a.bias != nullptr, load_bias(a.bias, a.bias_type, n), a.relu != 0));
        }
}

static int element_size(int type) { return type == NPA_FLOAT32 ? 4 : type == NPA_FLOAT16 || type == NPA_BFLOAT16 ? 2 : 1; }
static long long round16(long long v) { return (v + 15) / 16 * 16; }

template <typename F>
static void by_type(int type, F f) {
    if (type == NPA_FLOAT32) f(float());
    else if (type == NPA_FLOAT16) f(__half());
    else f(__nv_bfloat16());
}

static bool is_float(int type) { return type == NPA_FLOAT32 || type == NPA_FLOAT16 || type == NPA_BFLOAT16; }
static bool is_code(int type) { return type == NPA_INT8 || type == NPA_UINT8; }

static int launch_quantize(const void *x, int type, long long pitch, long long rows, int cols, bool is_unsigned, void *codes, long long codes_pitch,
                           float *scales, cudaStream_t st) {
    const long long blocks = (rows + 7) / 8;
    by_type(type, [&](auto t) {
        using T = decltype(t);
        launch_early(is_unsigned ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, (unsigned)blocks, 256, 0, st, static_cast<const T *>(x),
                     pitch, rows, cols, static_cast<uint8_t *>(codes), codes_pitch, scales);
    });
    return check_launch("quantize_rows_kernel");
}

static int launch_product(const Int8Args &a, int out_type, cudaStream_t st) {
    const dim3 grid((unsigned)((a.rows + kTileM - 1) / kTileM), (a.out_dim + kTileN - 1) / kTileN);
    by_type(out_type, [&](auto t) { launch_early(int8_tile_kernel<decltype(t)>, grid, 256, 0, st, a); });
    return check_launch("int8_tile_kernel");
}

static int check_rows(const char *me, int64_t rows, int32_t cols) {
    if (rows <= 0 || cols <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows and columns must be positive", me);
    if (rows > ((int64_t)1 << 31) - 1) return fail(NPA_ERR_UNSUPPORTED, "%s: supports fewer than 2^31 rows, got %lld", me, (long long)rows);
    return NPA_OK;
}

}  // namespace npa

using namespace npa;

extern "C" {

int npa_quantize_rows(const void *x, int32_t x_type, int64_t x_pitch, int64_t rows, int32_t cols, void *codes, int32_t codes_type, int64_t codes_pitch,
                      float *scales, void *stream) {
    const char *me = "npa_quantize_rows";
    const int rc = check_rows(me, rows, cols);
    if (rc != NPA_OK) return rc;
    if (!is_float(x_type) || !is_code(codes_type)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: x must be of a floating type, codes of an 8-bit one", me);
    if (!x || !codes || !scales) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: x, codes and scales must be non-NULL", me);
    if ((uintptr_t)x % element_size(x_type) || (uintptr_t)scales % 4) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: x and scales must be aligned to their types", me);
    if (x_pitch < 0 || codes_pitch < cols) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: the rows of codes overlap", me);
    return launch_quantize(x, x_type, x_pitch, rows, cols, codes_type == NPA_UINT8, codes, codes_pitch, scales, (cudaStream_t)stream);
}

int npa_dequantize_rows(const void *codes, int32_t codes_type, int64_t codes_pitch, const float *scales, int64_t rows, int32_t cols, void *out,
                        int32_t out_type, void *stream) {
    const char *me = "npa_dequantize_rows";
    const int rc = check_rows(me, rows, cols);
    if (rc != NPA_OK) return rc;
    if (!is_float(out_type) || !is_code(codes_type)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: out must be of a floating type, codes of an 8-bit one", me);
    if (!codes || !out || !scales) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: codes, scales and out must be non-NULL", me);
    if ((uintptr_t)out % element_size(out_type) || (uintptr_t)scales % 4) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: out and scales must be aligned to their types", me);
    if (codes_pitch < 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: codes_pitch must not be negative", me);
    const unsigned blocks = (unsigned)((rows + 7) / 8);
    by_type(out_type, [&](auto t) {
        using T = decltype(t);
        if (codes_type == NPA_UINT8)
            launch_early(dequantize_rows_kernel<T, uint8_t>, blocks, 256, 0, (cudaStream_t)stream, static_cast<const uint8_t *>(codes), codes_pitch, scales, rows,
                         cols, static_cast<T *>(out));
        else
            launch_early(dequantize_rows_kernel<T, int8_t>, blocks, 256, 0, (cudaStream_t)stream, static_cast<const int8_t *>(codes), codes_pitch, scales, rows,
                         cols, static_cast<T *>(out));
    });
    return check_launch("dequantize_rows_kernel");
}

static int64_t code_bytes(int64_t rows, int32_t cols) { return rows * round16(cols) + round16(rows * 4); }

int64_t npa_linear_int8_scratch_bytes(int32_t x_type, int64_t rows, int32_t in_dim) {
    if (rows <= 0 || in_dim <= 0 || is_code(x_type)) return 0;
    return code_bytes(rows, in_dim);
}

int npa_linear_int8(const void *x, int32_t x_type, int64_t x_pitch, const float *x_scales, const void *w, int64_t w_pitch, const float *w_scales,
                    const void *bias, int32_t bias_type, int32_t relu, void *out, int32_t out_type, int64_t rows, int32_t in_dim, int32_t out_dim,
                    void *scratch, int64_t scratch_bytes, void *stream) {
    const char *me = "npa_linear_int8";
    int rc = check_rows(me, rows, in_dim);
    if (rc != NPA_OK) return rc;
    if (out_dim <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: out_dim must be positive", me);
    if (in_dim > kInt8MaxIn) return fail(NPA_ERR_UNSUPPORTED, "%s: sums of up to %d products fit 32 bits, got in_dim %d", me, kInt8MaxIn, in_dim);
    if (!(is_float(x_type) || is_code(x_type)) || !is_float(out_type) || (bias && !is_float(bias_type)))
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: unknown type", me);
    if (!x || !w || !w_scales || !out) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: x, w, w_scales and out must be non-NULL", me);
    if ((uintptr_t)x % element_size(x_type) || (uintptr_t)out % element_size(out_type) || (bias && (uintptr_t)bias % element_size(bias_type)) ||
        ((uintptr_t)w_scales | (uintptr_t)x_scales) % 4)
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be aligned to its type", me);
    if (x_pitch < 0 || w_pitch < 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: pitches must not be negative", me);
    Int8Args a = {};
    a.w = static_cast<const int8_t *>(w); a.w_pitch = w_pitch; a.w_scales = w_scales; a.bias = bias; a.bias_type = bias_type; a.relu = relu;
    a.out = out; a.rows = rows; a.in = in_dim; a.out_dim = out_dim; a.x_unsigned = x_type == NPA_UINT8;
    if (is_code(x_type)) {
        if (!x_scales) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows of codes come with their scales", me);
        a.x = static_cast<const uint8_t *>(x); a.x_pitch = x_pitch; a.x_scales = x_scales;
    } else {
        const int64_t need = npa_linear_int8_scratch_bytes(x_type, rows, in_dim);
        if (!scratch || (uintptr_t)scratch % 16) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: scratch must be there, 16-byte aligned", me);
        if (scratch_bytes < need) return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, (long long)need);
        float *scales = reinterpret_cast<float *>(static_cast<char *>(scratch) + rows * round16(in_dim));
        rc = launch_quantize(x, x_type, x_pitch, rows, in_dim, false, scratch, round16(in_dim), scales, (cudaStream_t)stream);
        if (rc != NPA_OK) return rc;
        a.x = static_cast<const uint8_t *>(scratch); a.x_pitch = round16(in_dim); a.x_scales = scales;
    }
    return launch_product(a, out_type, (cudaStream_t)stream);
}

int64_t npa_mlp_int8_scratch_bytes(int64_t rows, int32_t in_dim, int32_t hidden, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || hidden <= 0 || out_dim <= 0) return 0;
    return code_bytes(rows, in_dim) + code_bytes(rows, hidden) + round16(rows * hidden * 4);
}

int npa_mlp_int8(const float *z, int64_t z_pitch, const void *w1, int64_t w1_pitch, const float *w1_scales, const float *b1, const void *w2, int64_t w2_pitch,
                 const float *w2_scales, float *y, int64_t rows, int32_t in_dim, int32_t hidden, int32_t out_dim, void *scratch, int64_t scratch_bytes,
                 void *stream) {
    const char *me = "npa_mlp_int8";
    int rc = check_rows(me, rows, in_dim);
    if (rc != NPA_OK) return rc;
    if (hidden <= 0 || out_dim <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: hidden and out_dim must be positive", me);
    if (!z || !w1 || !w1_scales || !b1 || !w2 || !w2_scales || !y) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be there", me);
    const int64_t need = npa_mlp_int8_scratch_bytes(rows, in_dim, hidden, out_dim);
    if (need && (!scratch || (uintptr_t)scratch % 16)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: scratch must be there, 16-byte aligned", me);
    if (scratch_bytes < need) return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, (long long)need);
    char *p = static_cast<char *>(scratch);
    float *h = reinterpret_cast<float *>(p + code_bytes(rows, in_dim) + code_bytes(rows, hidden));
    char *codes = p + code_bytes(rows, in_dim);
    float *scales = reinterpret_cast<float *>(codes + rows * round16(hidden));
    rc = npa_linear_int8(z, NPA_FLOAT32, z_pitch, nullptr, w1, w1_pitch, w1_scales, b1, NPA_FLOAT32, 1, h, NPA_FLOAT32, rows, in_dim, hidden, p,
                         code_bytes(rows, in_dim), stream);
    if (rc != NPA_OK) return rc;
    rc = launch_quantize(h, NPA_FLOAT32, hidden, rows, hidden, true, codes, round16(hidden), scales, (cudaStream_t)stream);
    if (rc != NPA_OK) return rc;
    return npa_linear_int8(codes, NPA_UINT8, round16(hidden), scales, w2, w2_pitch, w2_scales, nullptr, 0, 0, y, NPA_FLOAT32, rows, hidden, out_dim, nullptr, 0,
                           stream);
}

}  // extern "C"
