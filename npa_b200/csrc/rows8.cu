// Activations into 8 bits and back (rows8.cuh).  Reading and writing memory is all there has to be to either way; what bounds
// them is the instructions: of 8,191 x 4,100 bf16 (101 MB, 15.4 us) 26 us into 8 bits with 71 % of the issue slots taken, 30 us back with 67 %.
#include "rows8.cuh"

namespace npa {

// Rows whose addresses are multiples of W = 16 or 8 bytes: a thread takes eight values, four neighbours a group.
template <typename T, int W>
__global__ void __launch_bounds__(256) rows8_compress_kernel(const T *__restrict__ x, long long pitch, long long rows, int cols, int8_t *__restrict__ codes,
                                                             long long codes_pitch, uint8_t *__restrict__ exps) {
    after_previous_kernel();
    const int groups = rows8_groups(cols), each = 4 * groups;
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x, row = (rows * each) >> 32 ? at / each : (long long)((unsigned)at / (unsigned)each);
    const int part = (int)(at - row * each), k = 8 * part;
    const int left = row < rows ? cols - k : 0;
    float v[8];
    load_values<T, 8, W>(x + (left > 0 ? row * pitch + k : 0), left, v);
    unsigned largest = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) largest = max(largest, magnitude(v[q]));
    largest = max(largest, __shfl_xor_sync(kFull, largest, 1));
    largest = max(largest, __shfl_xor_sync(kFull, largest, 2));
    if (row >= rows) return;
    const unsigned e = rows8_exponent(largest);
    const float to_units = rows8_to_units(e);
    unsigned code[8];
    rows8_codes<8>(v, e, to_units, code);
    if (left > 0) store_codes<8>(reinterpret_cast<uint8_t *>(codes) + row * codes_pitch + k, left, (reinterpret_cast<uintptr_t>(codes) | codes_pitch) % 8 == 0, code);
    if (part % 4 == 0) exps[row * groups + part / 4] = (uint8_t)e;
}

// Other rows: a warp takes eight groups that follow one another, lane = column, so that its loads are lines and the maxima share their
// shuffles.  The codes leave through shared memory in pieces of 16 bytes (`whole`: where a row's pitch is its
// length rounded up to 16; in a wider one what follows a row stays as it was, and they leave as bytes):
// a store of 32 single bytes costs 12 clocks of an SM, whatever it hits (95 us for 8,191 rows of 4,100 bf16).  These rows by vectors 31.6 us,
// by lanes 69.6 (L2 flushed); 32,768 rows of 66 32-bit values 9.2 and 13.2: vectors where the addresses allow.
constexpr int kRowsFlight = 8;
template <typename T>
__global__ void __launch_bounds__(256) rows8_compress_lanes_kernel(const T *__restrict__ x, long long pitch, long long rows, int cols,
                                                                   int8_t *__restrict__ codes, long long codes_pitch, uint8_t *__restrict__ exps, int whole) {
    after_previous_kernel();
    __shared__ __align__(16) uint8_t staged[8][kRowsFlight * kRowsGroup];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = rows8_groups(cols);
    const long long first = ((long long)blockIdx.x * 8 + warp) * kRowsFlight, units = rows * groups;
    if (first >= units) return;
    const long long row0 = units >> 32 ? first / groups : (long long)((unsigned)first / (unsigned)groups);
    const int g0 = (int)(first - row0 * groups);
    float v[kRowsFlight];
    unsigned largest[kRowsFlight];
    long long row = row0;
    int g = g0;
#pragma unroll
    for (int i = 0; i < kRowsFlight; ++i) {
        const int k = g * kRowsGroup + lane;
        v[i] = row < rows && k < cols ? as_float(x[row * pitch + k]) : 0.f;
        largest[i] = magnitude(v[i]);
        if (++g == groups) {
            g = 0;
            ++row;
        }
    }
    const unsigned e = rows8_exponent(gather_max8(largest));  // of group lane / 4
    const float to_units = rows8_to_units(e);
    const int mine = lane >> 2;
    if ((lane & 3) == 0 && first + mine < units) exps[first + mine] = (uint8_t)e;
    uint8_t *to = staged[warp];
    row = row0;
    g = g0;
    const bool far = __any_sync(kFull, e >= 254u);
#pragma unroll
    for (int i = 0; i < kRowsFlight; ++i) {
        const float units_of = __shfl_sync(kFull, to_units, 4 * i);
        int code = (int)__float_as_uint(__fmaf_rn(v[i], units_of, kRoundWhole));
        if (far) code = rows8_code(v[i], units_of);
        if (whole) {
            to[i * kRowsGroup + lane] = (uint8_t)code;
        } else {
            const int k = g * kRowsGroup + lane;
            if (row < rows && k < cols) codes[row * codes_pitch + k] = (int8_t)code;
            if (++g == groups) {
                g = 0;
                ++row;
            }
        }
    }
    if (!whole) return;
    __syncwarp();
    // half a group a lane: 16 bytes, unless they lie behind the row's last column
    const long long at = first + (lane >> 1);
    if (lane < 2 * kRowsFlight && at < units) {
        const int ahead = g0 + (lane >> 1);
        const long long r = row0 + ahead / groups;
        const int k = (ahead % groups) * kRowsGroup + 16 * (lane & 1);
        if (k < cols) *reinterpret_cast<uint4 *>(codes + r * codes_pitch + k) = *reinterpret_cast<const uint4 *>(to + 16 * lane);
    }
}

template <typename T>
__device__ __forceinline__ T restored(float v) { return from_float<T>(v); }
template <>
__device__ __forceinline__ __half restored<__half>(float v) {  // the largest numbers may round to one above them in 8 bits
    return __float2half_rn(fabsf(v) > 65504.f ? copysignf(65504.f, v) : v);
}

// A thread writes 16 bytes, wherever in a row they lie (rows of an odd number of columns follow one another without a gap).
template <typename T>
__global__ void __launch_bounds__(256) rows8_restore_kernel(const int8_t *__restrict__ codes, long long codes_pitch, const uint8_t *__restrict__ exps,
                                                            long long rows, int cols, T *__restrict__ out) {
    after_previous_kernel();
    constexpr int V = 16 / sizeof(T);
    const long long first = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * V, total = rows * cols;
    if (first >= total) return;
    const int groups = rows8_groups(cols);
    long long row = total >> 32 ? first / cols : (long long)((unsigned)first / (unsigned)cols);
    int k = (int)(first - row * cols);
    union {
        uint4 quad;
        T value[V];
    } u;
    const int8_t *c = codes + row * codes_pitch;
    const uint8_t *e = exps + row * groups;
    if (k + V <= cols) {  // within one row: one group, or two
        const int g = k / kRowsGroup, left = (g + 1) * kRowsGroup - k;
        const float one = rows8_unit(e[g]), two = left < V ? rows8_unit(e[g + 1]) : one;
        unsigned word[V / 4];
        if (reinterpret_cast<uintptr_t>(c + k) % 4 == 0) {
#pragma unroll
            for (int w = 0; w < V / 4; ++w) word[w] = *reinterpret_cast<const unsigned *>(c + k + 4 * w);
        } else {
#pragma unroll
            for (int w = 0; w < V / 4; ++w) {
                const uint8_t *b = reinterpret_cast<const uint8_t *>(c + k + 4 * w);
                word[w] = (unsigned)b[0] | (unsigned)b[1] << 8 | (unsigned)b[2] << 16 | (unsigned)b[3] << 24;
            }
        }
#pragma unroll
        for (int w = 0; w < V / 4; ++w) {
            float v[4];
            rows8_numbers(word[w], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) u.value[4 * w + i] = restored<T>(v[i] * (4 * w + i < left ? one : two));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u.value[i] = row < rows ? restored<T>((float)c[k] * rows8_unit(e[k / kRowsGroup])) : T();
            if (++k == cols) {
                k = 0;
                ++row;
                c += codes_pitch;
                e += groups;
            }
        }
    }
    if (first + V <= total && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
        *reinterpret_cast<uint4 *>(out + first) = u.quad;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (first + i < total) out[first + i] = u.value[i];
    }
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
    if (cols > 1 << 30) return fail(NPA_ERR_UNSUPPORTED, "%s: supports up to 2^30 columns, got %d", me, (int)cols);
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
    by_float_type(type, [&](auto t) {
        using T = decltype(t);
        const uintptr_t lie = (uintptr_t)x | (uintptr_t)(x_pitch * (int64_t)sizeof(T));
        const bool vectors = lie % 8 == 0;
        const long long units = rows * rows8_groups(cols), blocks = vectors ? (4 * units + 255) / 256 : (units + 8 * kRowsFlight - 1) / (8 * kRowsFlight);
        const int whole = (uintptr_t)codes % 16 == 0 && codes_pitch == (cols + 15) / 16 * 16;
        if (vectors)
            launch_early(lie % 16 == 0 ? rows8_compress_kernel<T, 16> : rows8_compress_kernel<T, 8>, (unsigned)blocks, 256, 0, (cudaStream_t)stream, static_cast<const T *>(x), x_pitch, rows, cols,
                         static_cast<int8_t *>(codes), codes_pitch, exponents);
        else
            launch_early(rows8_compress_lanes_kernel<T>, (unsigned)blocks, 256, 0, (cudaStream_t)stream, static_cast<const T *>(x), x_pitch, rows, cols,
                         static_cast<int8_t *>(codes), codes_pitch, exponents, whole);
    });
    return check_launch("rows8_compress_kernel");
}

int npa_rows8_restore(const void *codes, int64_t codes_pitch, const uint8_t *exponents, int64_t rows, int32_t cols, void *out, int32_t type, void *stream) {
    const char *me = "npa_rows8_restore";
    const int rc = check_rows8(me, out, type, codes, exponents, rows, cols, codes_pitch);
    if (rc != NPA_OK) return rc;
    by_float_type(type, [&](auto t) {
        using T = decltype(t);
        const long long threads = (rows * cols * (int64_t)sizeof(T) + 15) / 16;
        launch_early(rows8_restore_kernel<T>, (unsigned)((threads + 255) / 256), 256, 0, (cudaStream_t)stream, static_cast<const int8_t *>(codes), codes_pitch,
                     exponents, rows, cols, static_cast<T *>(out));
    });
    return check_launch("rows8_restore_kernel");
}

}  // extern "C"
