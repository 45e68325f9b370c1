// Activations into 8 bits and back (rows8.cuh), and the adaptation MLP whose backward reads its input that way.
//
//     forward    y = relu(z W1^T + b1) W2^T                       keeps codes(z) and the bits of h > 0
//     backward   h = bits * (restore(codes) W1^T + b1)            dh = bits * (dy W2)
//                dz = dh W1,  dW1 = dh^T restore(codes),  db1 = sum of dh,  dW2 = dy^T h
//
// 1 + 1/32 byte per input and 16 bytes for the hidden layer instead of 4 per input and 512.  dz and db1 are those of the 32-bit
// backward, because the bits are those of the forward; dW1 and dW2 see the rounding of z to codes.
#include "rows8.cuh"

namespace npa {

constexpr int kMaskHidden = 128;

template <typename T>
__global__ void __launch_bounds__(256) rows8_compress_kernel(const T *__restrict__ x, long long pitch, long long rows, int cols, int8_t *__restrict__ codes,
                                                             long long codes_pitch, uint8_t *__restrict__ exps) {
    after_previous_kernel();
    const int lane = threadIdx.x & 31, groups = rows8_groups(cols);
    const long long unit = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);  // a warp per group
    if (unit >= rows * groups) return;
    const long long row = unit / groups;
    const int g = (int)(unit - row * groups), k = g * kRowsGroup + lane;
    const float v = k < cols ? as_float(x[row * pitch + k]) : 0.f;
    const unsigned e = rows8_exponent(warp_max(magnitude(v)));
    if (k < cols) codes[row * codes_pitch + k] = (int8_t)rows8_code(v, rows8_to_units(e));
    if (lane == 0) exps[unit] = (uint8_t)e;
}

template <typename T>
__device__ __forceinline__ T restored(float v) { return from_float<T>(v); }
template <>
__device__ __forceinline__ __half restored<__half>(float v) {  // the largest numbers may round to one above them in 8 bits
    return __float2half_rn(fabsf(v) > 65504.f ? copysignf(65504.f, v) : v);
}

template <typename T>
__global__ void __launch_bounds__(256) rows8_restore_kernel(const int8_t *__restrict__ codes, long long codes_pitch, const uint8_t *__restrict__ exps,
                                                            long long rows, int cols, T *__restrict__ out) {
    after_previous_kernel();
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= rows * cols) return;
    const long long row = at / cols;
    const int k = (int)(at - row * cols);
    out[at] = restored<T>((float)codes[row * codes_pitch + k] * rows8_unit(exps[row * rows8_groups(cols) + k / kRowsGroup]));
}

// Bits of h > 0: unit 32 w + i is bit i of word w.
__global__ void __launch_bounds__(256) mask_bits_kernel(const float *__restrict__ h, long long rows, unsigned *__restrict__ mask) {
    after_previous_kernel();
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const unsigned bits = __ballot_sync(kFull, at < rows * kMaskHidden && h[at] > 0.f);
    if ((threadIdx.x & 31) == 0 && at < rows * kMaskHidden) mask[at / 32] = bits;
}
__global__ void __launch_bounds__(256) apply_mask_kernel(float *__restrict__ a, float *__restrict__ b, long long rows, const unsigned *__restrict__ mask) {
    after_previous_kernel();
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= rows * kMaskHidden || (mask[at / 32] >> (at % 32) & 1u)) return;
    a[at] = 0.f;
    b[at] = 0.f;
}

template <typename F>
static void by_float_type(int type, F f) {
    if (type == NPA_FLOAT32) f(float());
    else if (type == NPA_FLOAT16) f(__half());
    else f(__nv_bfloat16());
}
static int float_size(int type) { return type == NPA_FLOAT32 ? 4 : type == NPA_FLOAT16 || type == NPA_BFLOAT16 ? 2 : 0; }

static int check_rows8(const char *me, const void *floats, int type, const void *codes, const void *exps, int64_t rows, int32_t cols, int64_t codes_pitch) {
    if (rows <= 0 || cols <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows and columns must be positive", me);
    if (rows * (int64_t)rows8_groups(cols) >= (int64_t)1 << 33 || rows * (int64_t)cols >= (int64_t)1 << 38)
        return fail(NPA_ERR_UNSUPPORTED, "%s: supports fewer than 2^33 groups and 2^38 values", me);
    if (!float_size(type)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: unknown type", me);
    if (!floats || !codes || !exps) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be non-NULL", me);
    if ((uintptr_t)floats % float_size(type)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: the values must be aligned to their type", me);
    if (codes_pitch < cols) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: the rows of codes overlap", me);
    return NPA_OK;
}

}  // namespace npa

using namespace npa;

extern "C" {

int npa_rows8_compress(const void *x, int32_t type, int64_t x_pitch, int64_t rows, int32_t cols, void *codes, int64_t codes_pitch, uint8_t *exponents,
                       void *stream) {
    const char *me = "npa_rows8_compress";
    const int rc = check_rows8(me, x, type, codes, exponents, rows, cols, codes_pitch);
    if (rc != NPA_OK) return rc;
    if (x_pitch < 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: x_pitch must not be negative", me);
    const long long units = rows * rows8_groups(cols);
    by_float_type(type, [&](auto t) {
        launch_early(rows8_compress_kernel<decltype(t)>, (unsigned)((units + 7) / 8), 256, 0, (cudaStream_t)stream, static_cast<const decltype(t) *>(x), x_pitch,
                     rows, cols, static_cast<int8_t *>(codes), codes_pitch, exponents);
    });
    return check_launch("rows8_compress_kernel");
}

int npa_rows8_restore(const void *codes, int64_t codes_pitch, const uint8_t *exponents, int64_t rows, int32_t cols, void *out, int32_t type, void *stream) {
    const char *me = "npa_rows8_restore";
    const int rc = check_rows8(me, out, type, codes, exponents, rows, cols, codes_pitch);
    if (rc != NPA_OK) return rc;
    by_float_type(type, [&](auto t) {
        launch_early(rows8_restore_kernel<decltype(t)>, (unsigned)((rows * cols + 255) / 256), 256, 0, (cudaStream_t)stream, static_cast<const int8_t *>(codes),
                     codes_pitch, exponents, rows, cols, static_cast<decltype(t) *>(out));
    });
    return check_launch("rows8_restore_kernel");
}

static int64_t round_floats(int64_t n) { return (n + 63) / 64 * 64; }

static int check_mlp8(const char *me, int64_t rows, int32_t in_dim, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || out_dim <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows, in_dim and out_dim must be positive", me);
    if (rows > ((int64_t)1 << 31) - 1 || in_dim > 175 || out_dim > 48)
        return fail(NPA_ERR_UNSUPPORTED, "%s: supports fewer than 2^31 rows, in <= 175 and out <= 48 (hidden width 128), got %lld, %d and %d", me, (long long)rows,
                    in_dim, out_dim);
    return NPA_OK;
}

int64_t npa_mlp_checkpoint_forward_scratch_bytes(int64_t rows, int32_t in_dim, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || out_dim <= 0) return 0;
    return npa_mlp_forward_tcgen05_scratch_bytes(in_dim, out_dim) + rows * kMaskHidden * 4;
}

int npa_mlp_checkpoint_forward(const float *z, const float *W1, const float *b1, const float *W2, float *y, int64_t rows, int32_t in_dim, int32_t out_dim,
                               int64_t w1_stride_out, int64_t w1_stride_in, int64_t w2_stride_out, int64_t w2_stride_in, void *codes, uint8_t *exponents,
                               uint32_t *mask, void *scratch, int64_t scratch_bytes, void *stream) {
    const char *me = "npa_mlp_checkpoint_forward";
    int rc = check_mlp8(me, rows, in_dim, out_dim);
    if (rc != NPA_OK) return rc;
    if (!z || !W1 || !b1 || !W2 || !y || !codes || !exponents || !mask) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be non-NULL", me);
    if (!scratch || ((uintptr_t)scratch | (uintptr_t)codes | (uintptr_t)mask) % 16)
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: codes, mask and scratch must be there, 16-byte aligned", me);
    const int64_t need = npa_mlp_checkpoint_forward_scratch_bytes(rows, in_dim, out_dim), image = npa_mlp_forward_tcgen05_scratch_bytes(in_dim, out_dim);
    if (scratch_bytes < need) return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, (long long)need);
    float *h = reinterpret_cast<float *>(static_cast<char *>(scratch) + image);
    rc = npa_mlp_forward_tcgen05(z, W1, b1, W2, h, y, rows, in_dim, out_dim, w1_stride_out, w1_stride_in, w2_stride_out, w2_stride_in, scratch, image, stream);
    if (rc != NPA_OK) return rc;
    launch_early(mask_bits_kernel, (unsigned)((rows * kMaskHidden + 255) / 256), 256, 0, (cudaStream_t)stream, h, rows, mask);
    if ((rc = check_launch("mask_bits_kernel")) != NPA_OK) return rc;
    return npa_rows8_compress(z, NPA_FLOAT32, in_dim, rows, in_dim, codes, rows8_pitch(in_dim), exponents, stream);
}

int64_t npa_mlp_checkpoint_backward_scratch_bytes(int64_t rows, int32_t in_dim, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || out_dim <= 0) return 0;
    return 4 * (round_floats(rows * in_dim) + 2 * round_floats(rows * kMaskHidden) + round_floats(npa_mlp_weight_grad_tcgen05_scratch_floats(rows, in_dim, out_dim))) +
           npa_linear_tcgen05_scratch_bytes(in_dim, kMaskHidden) + npa_linear_tcgen05_scratch_bytes(out_dim, kMaskHidden) +
           npa_linear_tcgen05_scratch_bytes(kMaskHidden, in_dim);
}

int npa_mlp_checkpoint_backward(const void *codes, const uint8_t *exponents, const uint32_t *mask, const float *W1, const float *b1, const float *W2,
                                const float *dy, float *dz, float *dW1, float *db1, float *dW2, int64_t rows, int32_t in_dim, int32_t out_dim,
                                int64_t w1_stride_out, int64_t w1_stride_in, int64_t w2_stride_out, int64_t w2_stride_in, void *scratch,
                                int64_t scratch_bytes, void *stream) {
    const char *me = "npa_mlp_checkpoint_backward";
    int rc = check_mlp8(me, rows, in_dim, out_dim);
    if (rc != NPA_OK) return rc;
    if (!codes || !exponents || !mask || !W1 || !b1 || !W2 || !dy) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every input must be non-NULL", me);
    if ((!dW1 || !db1 || !dW2) && (dW1 || db1 || dW2)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: dW1, db1 and dW2 come together", me);
    if (!scratch || ((uintptr_t)scratch | (uintptr_t)codes | (uintptr_t)mask | (uintptr_t)dy) % 16)
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: codes, mask, dy and scratch must be there, 16-byte aligned", me);
    const int64_t need = npa_mlp_checkpoint_backward_scratch_bytes(rows, in_dim, out_dim);
    if (scratch_bytes < need) return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, (long long)need);
    float *z = static_cast<float *>(scratch), *h = z + round_floats(rows * in_dim), *dh = h + round_floats(rows * kMaskHidden),
          *partial = dh + round_floats(rows * kMaskHidden);
    const int64_t floats = npa_mlp_weight_grad_tcgen05_scratch_floats(rows, in_dim, out_dim), i1 = npa_linear_tcgen05_scratch_bytes(in_dim, kMaskHidden),
                  i2 = npa_linear_tcgen05_scratch_bytes(out_dim, kMaskHidden), i3 = npa_linear_tcgen05_scratch_bytes(kMaskHidden, in_dim);
    char *image = reinterpret_cast<char *>(partial + round_floats(floats));
    if ((rc = npa_rows8_restore(codes, rows8_pitch(in_dim), exponents, rows, in_dim, z, NPA_FLOAT32, stream)) != NPA_OK) return rc;
    if ((rc = npa_linear_tcgen05(z, W1, b1, nullptr, h, rows, in_dim, kMaskHidden, w1_stride_out, w1_stride_in, 0, image, i1, stream)) != NPA_OK) return rc;
    if ((rc = npa_linear_tcgen05(dy, W2, nullptr, nullptr, dh, rows, out_dim, kMaskHidden, w2_stride_in, w2_stride_out, 0, image + i1, i2, stream)) != NPA_OK) return rc;
    launch_early(apply_mask_kernel, (unsigned)((rows * kMaskHidden + 255) / 256), 256, 0, (cudaStream_t)stream, h, dh, rows, mask);
    if ((rc = check_launch("apply_mask_kernel")) != NPA_OK) return rc;
    if (dz && (rc = npa_linear_tcgen05(dh, W1, nullptr, nullptr, dz, rows, kMaskHidden, in_dim, w1_stride_in, w1_stride_out, 0, image + i1 + i2, i3, stream)) != NPA_OK)
        return rc;
    if (!dW1) return NPA_OK;
    return npa_mlp_weight_grad_tcgen05(z, dh, h, dy, rows, in_dim, kMaskHidden, out_dim, partial, floats, dW1, dW2, db1, stream);
}

}  // extern "C"
