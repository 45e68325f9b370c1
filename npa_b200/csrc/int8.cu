// Products in 8-bit integers: rows quantised with a scale each, weights with a scale for each output channel.
//
//     out[m, n] = act( float(sum_k q[m, k] w[n, k]) * (s[m] * t[n]) + bias[n] )
//
// The sum is one of integers and exact (a chain of 65,536 products of 255 and 127 stays below 2^31); behind it are three roundings of
// 32 bits -- the product of the scales, its product with the sum, the bias -- and the one to the type of the output.
#include <type_traits>

#include "int8.cuh"
#include "ops.cuh"

namespace npa {

constexpr int kInt8MaxIn = 65536;

// ---- rows into codes -------------------------------------------------------------------------------------------------
// T threads per row, each with V neighbouring values at a time (16 to 32 bytes, where the rows' addresses allow; single values, so that
// a warp's loads are lines, where they do not), up to kQuantizeHeld of them kept in registers between the largest magnitude and the
// codes; what is beyond is read twice, the second time from L1 or L2.
constexpr int kQuantizeHeld = 4;

template <typename X, bool UNSIGNED, int T, int V, int W>
__global__ void __launch_bounds__(T > 128 ? T : 128) quantize_rows_kernel(const X *__restrict__ x, long long pitch, long long rows, int cols,
                                                                         uint8_t *__restrict__ codes, long long codes_pitch, float *__restrict__ scales) {
    after_previous_kernel();
    constexpr int kRows = T >= 128 ? 1 : 128 / T;
    const int t = threadIdx.x % T;
    const bool aligned = (reinterpret_cast<uintptr_t>(codes) | codes_pitch) % 8 == 0;
    // (in their own type: half the registers for 16 bits, and twice the rows under way)
    Values<X, V, W> held[kQuantizeHeld], next[kQuantizeHeld];
    auto load = [&](Values<X, V, W>(&to)[kQuantizeHeld], long long row) {
        const X *p = x + (row < rows ? row : 0) * pitch;
        const int end = row < rows ? cols : 0;
#pragma unroll
        for (int i = 0; i < kQuantizeHeld; ++i) to[i].load(p + (i * T + t) * V, end - (i * T + t) * V);
    };
    long long row = (long long)blockIdx.x * kRows + threadIdx.x / T;
    const long long step = (long long)gridDim.x * kRows;
    load(held, row);
    // (the block's rows end together: their threads share warps and barriers)
    for (int turn = 0; row - threadIdx.x / T < rows; row += step, turn ^= 1) {
        load(next, row + step);  // on its way meanwhile
        const bool here = row < rows;
        const X *p = x + (here ? row : 0) * pitch;
        const int end = here ? cols : 0;
        unsigned largest = 0;
#pragma unroll
        for (int i = 0; i < kQuantizeHeld; ++i) {
            float v[V];
            held[i].get(v);
#pragma unroll
            for (int q = 0; q < V; ++q) largest = max(largest, magnitude(quantizable<UNSIGNED>(v[q])));
        }
        for (int k = (kQuantizeHeld * T + t) * V; k < end; k += T * V) {
            float w[V];
            load_values<X, V, W>(p + k, end - k, w);
#pragma unroll
            for (int q = 0; q < V; ++q) largest = max(largest, magnitude(quantizable<UNSIGNED>(w[q])));
        }
        largest = warp_max<(T < 32 ? T : 32)>(largest);
        if constexpr (T > 32) {
            __shared__ unsigned most[2][T / 32];
            if (t % 32 == 0) most[turn][t / 32] = largest;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < T / 32; ++w) largest = max(largest, most[turn][w]);
        }
        if (here) {
            float inverse;
            const float scale = row_scale(largest, UNSIGNED ? 255.f : 127.f, inverse);
            uint8_t *out = codes + row * codes_pitch;
            auto put = [&](int k, const float (&w)[V]) {
                float x[V];
                unsigned code[V];
#pragma unroll
                for (int q = 0; q < V; ++q) x[q] = quantizable<UNSIGNED>(w[q]);
                if (inverse == 0.f) {  // the row is not finite
#pragma unroll
                    for (int q = 0; q < V; ++q) code[q] = 0;
                } else {
                    row_codes<V>(x, scale, inverse, code);
                }
                store_codes<V>(out + k, cols - k, aligned, code);
            };
#pragma unroll
            for (int i = 0; i < kQuantizeHeld; ++i)
                if ((i * T + t) * V < cols) {
                    float v[V];
                    held[i].get(v);
                    put((i * T + t) * V, v);
                }
            for (int k = (kQuantizeHeld * T + t) * V; k < cols; k += T * V) {
                float w[V];
                load_values<X, V, W>(p + k, cols - k, w);
                put(k, w);
            }
            if (t == 0) scales[row] = scale;
        }
#pragma unroll
        for (int i = 0; i < kQuantizeHeld; ++i) held[i] = next[i];
    }
}

// Rows of up to 32 kBlocks values whose addresses fit no vector: a warp takes eight of them, lane = column, so that its loads are lines
// and the maxima share their shuffles.  Codes leave through shared memory in 16 bytes a lane where a row's pitch is its length rounded up
// to 16 (`whole`: what lies between is the row's own); in a wider pitch what follows a row stays as it was.
template <typename X, bool UNSIGNED, int kBlocks>
__global__ void __launch_bounds__(128) quantize_lanes_kernel(const X *__restrict__ x, long long pitch, long long rows, int cols, uint8_t *__restrict__ codes,
                                                             long long codes_pitch, float *__restrict__ scales) {
    after_previous_kernel();
    __shared__ __align__(16) uint8_t staged[4][8][32 * kBlocks];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row0 = ((long long)blockIdx.x * 4 + warp) * 8;
    if (row0 >= rows) return;
    float v[8][kBlocks];
    unsigned largest[8];
    const int there = rows - row0 < 8 ? (int)(rows - row0) : 8;
    const bool whole = reinterpret_cast<uintptr_t>(codes) % 16 == 0 && codes_pitch == (cols + 15) / 16 * 16;
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) v[r][b] = r < there && 32 * b + lane < cols ? quantizable<UNSIGNED>(as_float(x[(row0 + r) * pitch + 32 * b + lane])) : 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        largest[r] = 0;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) largest[r] = max(largest[r], magnitude(v[r][b]));
    }
    float back;
    const float own = row_scale(gather_max8(largest), UNSIGNED ? 255.f : 127.f, back);  // four lanes a row
    if (lane % 4 == 0 && lane / 4 < there) scales[row0 + lane / 4] = own;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const float scale = __shfl_sync(kFull, own, 4 * r), inverse = __shfl_sync(kFull, back, 4 * r);
        unsigned code[kBlocks];
        row_codes<kBlocks>(v[r], scale, inverse, code);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const uint8_t c = inverse == 0.f ? (uint8_t)0 : (uint8_t)code[b];
            if (whole) staged[warp][r][32 * b + lane] = c;
            else if (r < there && 32 * b + lane < cols) codes[(row0 + r) * codes_pitch + 32 * b + lane] = c;
        }
    }
    if (!whole) return;
    __syncwarp();
    const int pieces = (cols + 15) / 16;
    for (int q = lane; q < there * pieces; q += 32) {
        const int r = q / pieces, k = 16 * (q - r * pieces);
        *reinterpret_cast<uint4 *>(codes + (row0 + r) * codes_pitch + k) = *reinterpret_cast<const uint4 *>(&staged[warp][r][k]);
    }
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

// ---- few rows --------------------------------------------------------------------------------------------------------
// Up to 16 rows (a token, a handful of particles): the weights are read once, from memory or L2, and that is the time.  Each block holds
// the codes of all rows in shared memory.  It quantises up to 4,096 values itself; of more, every block does too much of the same, and a
// launch in front does it (us inside / in front, weights in L2: 1 x 1,024 3.7 / 4.8, 1 x 4,096 5.8 / 5.9, 8 x 1,024 8.1 / 5.6,
// 4 x 4,096 13.2 / 7.7).  Against the tensor cores' kernel, us (this / that): 1 x 4,096 x 4,096 5.8 / 18.5, 8 10.7 / 18.2, 16 16.1 / 17.6;
// 16 x 1,024 x 1,024 6.9 / 8.1, 16 x 2,048 x 5,120 13.7 / 11.9: 16 rows is where they meet.
// a warp takes NC channels and a lane 16 bytes of each at a time, NC x 4 loads in flight; four dp4a per row and 16 bytes are free
// beside them.  Where the channels alone would not fill the SMs, the warps of a block share a channel's length.
constexpr int kFewRows = 16, kFewBytes = 96 * 1024, kFewWarps = 8, kFewQuantized = 4096;

template <bool UNSIGNED>
__device__ __forceinline__ int dot4(unsigned x, unsigned w, int acc) {
    if constexpr (UNSIGNED) asm("dp4a.u32.s32 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(w));
    else acc = __dp4a((int)x, (int)w, acc);
    return acc;
}
// 16 weights of which `left` exist.
__device__ __forceinline__ uint4 load_weights(const int8_t *p, int left) {
    if (left >= 16) return __ldg(reinterpret_cast<const uint4 *>(p));
    unsigned v[4] = {};
#pragma unroll
    for (int q = 0; q < 15; ++q)
        if (q < left) v[q / 4] |= (unsigned)(uint8_t)__ldg(p + q) << (8 * (q % 4));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// The codes and scales of all rows into shared memory; every thread of the block.
template <int ROWS>
__device__ __forceinline__ void few_rows_codes(const Int8Args &a, uint8_t *codes, int pitch, float *scales) {
    const int rows = (int)a.rows, K = a.in;
    if (a.x_type >= NPA_INT8) {
        const uint8_t *x = static_cast<const uint8_t *>(a.x);
        if ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)a.x_pitch) % 16 == 0 && a.x_pitch >= pitch) {  // (codes behind a row's end meet weights of zero)
            const int pieces = pitch / 16;
            for (int q = threadIdx.x; q < ROWS * pieces; q += kFewWarps * 32) {
                const int r = q / pieces, k = 16 * (q - r * pieces);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < rows && k + 16 <= K) {
                    v = __ldg(reinterpret_cast<const uint4 *>(x + r * a.x_pitch + k));
                } else if (r < rows) {
                    unsigned w[4] = {};
#pragma unroll
                    for (int j = 0; j < 15; ++j)
                        if (k + j < K) w[j / 4] |= (unsigned)__ldg(x + r * a.x_pitch + k + j) << (8 * (j % 4));
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
                *reinterpret_cast<uint4 *>(codes + r * pitch + k) = v;
            }
        } else {
            for (int q = threadIdx.x; q < ROWS * pitch; q += kFewWarps * 32) {
                const int r = q / pitch, k = q - r * pitch;
                codes[q] = r < rows && k < K ? __ldg(x + r * a.x_pitch + k) : 0;
            }
        }
        if (threadIdx.x < ROWS) scales[threadIdx.x] = threadIdx.x < rows ? __ldg(a.x_scales + threadIdx.x) : 0.f;
        return;
    }
    __shared__ unsigned most[ROWS];
    if (threadIdx.x < ROWS) most[threadIdx.x] = 0;
    __syncthreads();
    auto pass = [&](auto *x, bool vectors, auto use) {  // use(row, column, values, how many)
        using X = std::remove_cv_t<std::remove_pointer_t<decltype(x)>>;
        if (vectors) {
            const int chunks = (K + 7) / 8;
            for (int q = threadIdx.x; q < rows * chunks; q += kFewWarps * 32) {
                const int r = q / chunks, k = 8 * (q - r * chunks);
                float v[8];
                load_values<X, 8>(x + r * a.x_pitch + k, K - k, v);
                use(r, k, v, 8);
            }
        } else {
            for (int q = threadIdx.x; q < rows * K; q += kFewWarps * 32) {
                const int r = q / K, k = q - r * K;
                float v[8];
                v[0] = as_float(x[r * a.x_pitch + k]);
                use(r, k, v, 1);
            }
        }
    };
    auto both = [&](auto *x) {
        const bool vectors = (reinterpret_cast<uintptr_t>(x) | (uintptr_t)(a.x_pitch * (long long)sizeof(*x))) % 16 == 0;
        int row = -1;
        unsigned largest = 0;
        pass(x, vectors, [&](int r, int, const float(&v)[8], int n) {
            if (r != row) {
                if (row >= 0) atomicMax(&most[row], largest);
                row = r;
                largest = 0;
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < n) largest = max(largest, magnitude(v[q]));
        });
        // threads of a warp mostly hold the same row: one atomic then
        const int first = __shfl_sync(kFull, row, 0);
        if (__all_sync(kFull, row == first)) {
            largest = warp_max(largest);
            if (row >= 0 && threadIdx.x % 32 == 0) atomicMax(&most[row], largest);
        } else if (row >= 0) {
            atomicMax(&most[row], largest);
        }
        __syncthreads();
        pass(x, vectors, [&](int r, int k, const float(&v)[8], int n) {
            float inverse;
            const float scale = row_scale(most[r], 127.f, inverse);
            unsigned w[2] = {};
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < n) w[q / 4] |= ((unsigned)row_code(v[q], scale, inverse) & 0xffu) << (8 * (q % 4));
            if (n == 8) *reinterpret_cast<uint2 *>(codes + r * pitch + k) = make_uint2(w[0], w[1]);  // (what is not there is zero: so are its codes)
            else codes[r * pitch + k] = (uint8_t)w[0];
        });
    };
    // rows and columns that do not exist (a chunk of eight may end before the pitch does)
    for (int q = threadIdx.x; q < ROWS * 16; q += kFewWarps * 32) {
        const int r = q / 16, k = pitch - 16 + q % 16;
        if (r >= rows || k >= (K + 7) / 8 * 8 || k >= K) codes[r * pitch + k] = 0;
    }
    for (int q = threadIdx.x; q < (ROWS - rows) * (pitch / 16); q += kFewWarps * 32)
        *reinterpret_cast<uint4 *>(codes + rows * pitch + 16 * q) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (a.x_type == NPA_FLOAT32) both(static_cast<const float *>(a.x));
    else if (a.x_type == NPA_FLOAT16) both(static_cast<const __half *>(a.x));
    else both(static_cast<const __nv_bfloat16 *>(a.x));
    if (threadIdx.x < ROWS) {
        float inverse;
        scales[threadIdx.x] = row_scale(most[threadIdx.x], 127.f, inverse);
    }
}

template <int ROWS, int NC, bool UNSIGNED>
__global__ void __launch_bounds__(kFewWarps * 32) int8_few_rows_kernel(const __grid_constant__ Int8Args a, int share) {
    after_previous_kernel();
    extern __shared__ __align__(16) uint8_t few_codes[];
    __shared__ float scales[ROWS];
    __shared__ int sums[kFewWarps][NC * ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = (a.in + 15) / 16 * 16;
    const int part = warp % share;  // `share` warps divide the length of their channels
    const int n0 = (blockIdx.x * (kFewWarps / share) + warp / share) * NC;
    int acc[NC][ROWS] = {};
    const int8_t *w[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) w[c] = a.w + (long long)min(n0 + c, a.out_dim - 1) * a.w_pitch;
    const int step = 512 * share, full = n0 < a.out_dim ? a.in / 16 * 16 : 0;
    int k = (part * 32 + lane) * 16;
    // the first weights are on their way while the rows are quantised
    uint4 wv[4][NC];
    auto fetch = [&]() {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < NC; ++c) wv[u][c] = __ldg(reinterpret_cast<const uint4 *>(w[c] + k + u * step));
    };
    bool ahead = k + 3 * step < full;
    if (ahead) fetch();
    few_rows_codes<ROWS>(a, few_codes, pitch, scales);
    __syncthreads();
    if (n0 < a.out_dim) {
        auto add = [&](int k, const uint4(&wv)[NC]) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const uint4 xv = *reinterpret_cast<const uint4 *>(few_codes + r * pitch + k);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    acc[c][r] = dot4<UNSIGNED>(xv.x, wv[c].x, acc[c][r]);
                    acc[c][r] = dot4<UNSIGNED>(xv.y, wv[c].y, acc[c][r]);
                    acc[c][r] = dot4<UNSIGNED>(xv.z, wv[c].z, acc[c][r]);
                    acc[c][r] = dot4<UNSIGNED>(xv.w, wv[c].w, acc[c][r]);
                }
            }
        };
        while (ahead) {
#pragma unroll
            for (int u = 0; u < 4; ++u) add(k + u * step, wv[u]);
            k += 4 * step;
            ahead = k + 3 * step < full;
            if (ahead) fetch();
        }
        for (; k < a.in; k += step) {
            uint4 last[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) last[c] = load_weights(w[c] + k, a.in - k);
            add(k, last);
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int sum = __reduce_add_sync(kFull, acc[c][r]);
            if (lane == (c * ROWS + r) % 32) sums[warp][c * ROWS + r] = sum;
        }
    __syncthreads();
    if (part != 0 || n0 >= a.out_dim) return;
    for (int q = lane; q < NC * ROWS; q += 32) {
        const int c = q / ROWS, r = q % ROWS, n = n0 + c;
        if (r >= a.rows || n >= a.out_dim) continue;
        int sum = 0;
        for (int p = 0; p < share; ++p) sum += sums[warp + p][q];
        const float v = int8_value(sum, scales[r], __ldg(a.w_scales + n), a.bias != nullptr, a.bias ? load_value(a.bias, a.bias_type, n) : 0.f, a.relu != 0);
        const long long at = (long long)r * a.out_dim + n;
        if (a.out_type == NPA_FLOAT32) static_cast<float *>(a.out)[at] = v;
        else if (a.out_type == NPA_FLOAT16) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
        else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
    }
}

// ---- codes that the tensor cores cannot take as they lie ----------------------------------------------------------------
// Rows into a pitch of multiples of 16 bytes, unsigned codes shifted to the signed ones that the tensor cores are given (p - 128, which flips the
// top bit).
__global__ void __launch_bounds__(256) repack_codes_kernel(const uint8_t *__restrict__ from, long long from_pitch, long long rows, int cols, unsigned flip,
                                                           uint8_t *__restrict__ to, int to_pitch) {
    after_previous_kernel();
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x, row = at / to_pitch;
    const int k = (int)(at - row * to_pitch);
    if (row < rows) to[at] = k < cols ? (uint8_t)(from[row * from_pitch + k] ^ flip) : (uint8_t)0;
}
// What the shift takes from a channel's sum, divided by 128.
__global__ void __launch_bounds__(256) weight_sums_kernel(const int8_t *__restrict__ w, long long pitch, int rows, int cols, int *__restrict__ sums) {
    after_previous_kernel();
    const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    int sum = 0;
    for (int k = 16 * lane; k < cols; k += 512) {
        const uint4 v = load_weights(w + row * pitch + k, cols - k);
        sum = dot4<false>(0x01010101u, v.x, sum);
        sum = dot4<false>(0x01010101u, v.y, sum);
        sum = dot4<false>(0x01010101u, v.z, sum);
        sum = dot4<false>(0x01010101u, v.w, sum);
    }
    sum = __reduce_add_sync(kFull, sum);
    if (lane == 0) sums[row] = sum;
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

template <typename X, bool UNSIGNED, int T, int V, int W>
static void launch_quantize_shape(const void *x, long long pitch, long long rows, int cols, void *codes, long long codes_pitch, float *scales, cudaStream_t st) {
    constexpr int kRows = T >= 128 ? 1 : 128 / T, kThreads = T > 128 ? T : 128;
    const long long blocks = (rows + kRows - 1) / kRows;
    int resident = 0;  // (where it cannot be asked for, the launch says why)
    if (persistent_ctas(quantize_rows_kernel<X, UNSIGNED, T, V, W>, kThreads, 0, &resident) != NPA_OK) resident = 148;
    launch_early(quantize_rows_kernel<X, UNSIGNED, T, V, W>, (unsigned)(blocks < resident ? blocks : resident), kThreads, 0, st, static_cast<const X *>(x), pitch, rows,
                 cols, static_cast<uint8_t *>(codes), codes_pitch, scales);
}
template <typename X, bool UNSIGNED>
static void launch_quantize_type(const void *x, long long pitch, long long rows, int cols, void *codes, long long codes_pitch, float *scales, cudaStream_t st) {
#define NPA_QUANTIZE(T, V, W) launch_quantize_shape<X, UNSIGNED, T, V, W>(x, pitch, rows, cols, codes, codes_pitch, scales, st)
    const uintptr_t lie = (uintptr_t)x | (uintptr_t)(pitch * (long long)sizeof(X));
    if (lie % 16 == 0) {
        // the fewest threads whose registers hold a row.  Measured with 8, 32, 128, 256 of them, us (bf16, L2 flushed):
        //   32,768 x 256 14.4, 23.6, 66.6, 126;  8,192 x 1,024 23.6, 13.4, 23.6, 37.9;  8,192 x 4,096 104, 45.0, 29.7, 44.0;
        //   4,096 x 8,192 198, 54.2, 39.8, 29.7
        if (cols <= 256) NPA_QUANTIZE(8, 8, 16);
        else if (cols <= 1024) NPA_QUANTIZE(32, 8, 16);
        else if (cols <= 4096) NPA_QUANTIZE(128, 8, 16);
        else NPA_QUANTIZE(256, 8, 16);
    } else if (lie % 8 == 0) {
        if (cols <= 256) NPA_QUANTIZE(8, 8, 8);
        else if (cols <= 1024) NPA_QUANTIZE(32, 8, 8);
        else if (cols <= 4096) NPA_QUANTIZE(128, 8, 8);
        else NPA_QUANTIZE(256, 8, 8);
    } else {
        if (cols <= 512) {
            // (65,536 rows of 67, 163, 255 32-bit values: 14.3, 19.5, 25.6 us; by single values of 128 threads 52, 58, 60)
            void (*const kernel)(const X *, long long, long long, int, uint8_t *, long long, float *) =
                cols <= 64 ? quantize_lanes_kernel<X, UNSIGNED, 2> : cols <= 128 ? quantize_lanes_kernel<X, UNSIGNED, 4>
                : cols <= 192 ? quantize_lanes_kernel<X, UNSIGNED, 6> : cols <= 256 ? quantize_lanes_kernel<X, UNSIGNED, 8> : nullptr;
            if (kernel) {
                launch_early(kernel, (unsigned)((rows + 31) / 32), 128, 0, st, static_cast<const X *>(x), pitch, rows, cols, static_cast<uint8_t *>(codes), codes_pitch,
                             scales);
                return;
            }
            NPA_QUANTIZE(128, 1, 16);
        } else {
            NPA_QUANTIZE(256, 1, 16);
        }
    }
#undef NPA_QUANTIZE
}
static int launch_quantize(const void *x, int type, long long pitch, long long rows, int cols, bool is_unsigned, void *codes, long long codes_pitch,
                           float *scales, cudaStream_t st) {
    by_type(type, [&](auto t) {
        using X = decltype(t);
        if (is_unsigned) launch_quantize_type<X, true>(x, pitch, rows, cols, codes, codes_pitch, scales, st);
        else launch_quantize_type<X, false>(x, pitch, rows, cols, codes, codes_pitch, scales, st);
    });
    return check_launch("quantize_rows_kernel");
}

template <int ROWS, int NC>
static int launch_few_rows_shape(const Int8Args &a, int share, cudaStream_t st) {
    const auto kernel = a.x_type == NPA_UINT8 ? int8_few_rows_kernel<ROWS, NC, true> : int8_few_rows_kernel<ROWS, NC, false>;
    const int smem = ROWS * (int)round16(a.in), groups = (a.out_dim + NC - 1) / NC, each = kFewWarps / share;
    if (smem > 48 * 1024 - 2048) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewBytes);
        if (e != cudaSuccess) return fail(NPA_ERR_CUDA, "npa_linear_int8: raising the shared-memory limit: %s", cudaGetErrorString(e));
    }
    launch_early(kernel, (groups + each - 1) / each, kFewWarps * 32, smem, st, a, share);
    return check_launch("int8_few_rows_kernel");
}
static int padded_rows(long long rows) { return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }
static bool few_rows(long long rows, int in) { return rows <= kFewRows && padded_rows(rows) * round16(in) <= kFewBytes; }
static int launch_few_rows(const Int8Args &a, cudaStream_t st) {
    // four channels a warp where that still gives every SM its eight warps (1 x 2,048: 8,192 channels 15.4 -> 13.2 us, 4,096 the same; 8
    // rows, 4,096 channels 17.4 -> 13.3); the length shared where single channels do not (8,192 x 256: 15.4 us alone, 13.3 by two or
    // four, 15.2 by eight)
    const bool wide = a.out_dim >= 148 * kFewWarps * 2;
    int share = 1;
    while (!wide && share < kFewWarps && (long long)a.out_dim * share < 148 * kFewWarps && a.in > 512 * share) share *= 2;
    switch (padded_rows(a.rows)) {
        case 1: return wide ? launch_few_rows_shape<1, 4>(a, share, st) : launch_few_rows_shape<1, 1>(a, share, st);
        case 2: return wide ? launch_few_rows_shape<2, 4>(a, share, st) : launch_few_rows_shape<2, 1>(a, share, st);
        case 4: return wide ? launch_few_rows_shape<4, 4>(a, share, st) : launch_few_rows_shape<4, 1>(a, share, st);
        case 8: return wide ? launch_few_rows_shape<8, 2>(a, share, st) : launch_few_rows_shape<8, 1>(a, share, st);
        default: return wide ? launch_few_rows_shape<16, 2>(a, share, st) : launch_few_rows_shape<16, 1>(a, share, st);
    }
}

static int launch_repack(const void *from, long long from_pitch, long long rows, int cols, unsigned flip, void *to, cudaStream_t st) {
    const long long total = rows * round16(cols);
    launch_early(repack_codes_kernel, (unsigned)((total + 255) / 256), 256, 0, st, static_cast<const uint8_t *>(from), from_pitch, rows, cols, flip,
                 static_cast<uint8_t *>(to), (int)round16(cols));
    return check_launch("repack_codes_kernel");
}

static bool aligned_codes(const void *p, long long pitch) { return ((uintptr_t)p | (uintptr_t)pitch) % 16 == 0; }

// What a call needs beside its arguments: codes and scales of floating rows, or a copy of codes that do not lie as the kernels want
// them, a copy of such weights, sums of the channels' weights.
struct Int8Plan {
    bool few, quantize, repack_x, repack_w, sums;
    long long o_scales, o_w, o_sums, bytes;
    Int8Plan(const void *x, int x_type, long long x_pitch, const void *w, long long w_pitch, long long rows, int in, int out_dim) {
        few = few_rows(rows, in);
        quantize = is_float(x_type) && (!few || rows * in > kFewQuantized);
        repack_x = !few && is_code(x_type) && (x_type == NPA_UINT8 || !aligned_codes(x, x_pitch) || x_pitch < in);
        repack_w = !aligned_codes(w, w_pitch) || w_pitch < in;  // (rows that overlap: TMA wants none)
        sums = !few && x_type == NPA_UINT8;
        o_scales = quantize || repack_x ? rows * round16(in) : 0;
        o_w = o_scales + (quantize ? round16(rows * 4) : 0);
        o_sums = o_w + (repack_w ? (long long)out_dim * round16(in) : 0);
        bytes = o_sums + (sums ? round16((long long)out_dim * 4) : 0);
    }
};

static int check_rows(const char *me, int64_t rows, int32_t cols) {
    if (rows <= 0 || cols <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows and columns must be positive", me);
    if (rows > ((int64_t)1 << 31) - 1) return fail(NPA_ERR_UNSUPPORTED, "%s: supports fewer than 2^31 rows, got %lld", me, (long long)rows);
    if (cols > 1 << 30) return fail(NPA_ERR_UNSUPPORTED, "%s: supports up to 2^30 columns, got %d", me, (int)cols);
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

int64_t npa_linear_int8_scratch_bytes(const void *x, int32_t x_type, int64_t x_pitch, const void *w, int64_t w_pitch, int64_t rows, int32_t in_dim,
                                      int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || out_dim <= 0) return 0;
    return Int8Plan(x, x_type, x_pitch, w, w_pitch, rows, in_dim, out_dim).bytes;
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
    if (is_code(x_type) && !x_scales) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows of codes come with their scales", me);
    const Int8Plan plan(x, x_type, x_pitch, w, w_pitch, rows, in_dim, out_dim);
    if (plan.bytes && (!scratch || (uintptr_t)scratch % 16)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: scratch must be there, 16-byte aligned", me);
    if (scratch_bytes < plan.bytes)
        return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, plan.bytes);
    const cudaStream_t st = (cudaStream_t)stream;
    char *s = static_cast<char *>(scratch);
    Int8Args a = {};
    a.x = x; a.x_type = x_type; a.x_pitch = x_pitch; a.x_scales = x_scales; a.w = static_cast<const int8_t *>(w); a.w_pitch = w_pitch; a.w_scales = w_scales;
    a.bias = bias; a.bias_type = bias_type; a.relu = relu; a.out = out; a.out_type = out_type; a.rows = rows; a.in = in_dim; a.out_dim = out_dim;
    if (plan.repack_w) {
        if ((rc = launch_repack(w, w_pitch, out_dim, in_dim, 0, s + plan.o_w, st)) != NPA_OK) return rc;
        a.w = reinterpret_cast<const int8_t *>(s + plan.o_w); a.w_pitch = round16(in_dim);
    }
    if (plan.quantize) {
        float *scales = reinterpret_cast<float *>(s + plan.o_scales);
        if ((rc = launch_quantize(x, x_type, x_pitch, rows, in_dim, false, s, round16(in_dim), scales, st)) != NPA_OK) return rc;
        a.x_scales = scales;
    }
    if (plan.repack_x && (rc = launch_repack(x, x_pitch, rows, in_dim, x_type == NPA_UINT8 ? 0x80u : 0u, s, st)) != NPA_OK) return rc;
    if (plan.quantize || plan.repack_x) {
        a.x = s; a.x_pitch = round16(in_dim); a.x_type = NPA_INT8;
    }
    if (plan.few) return launch_few_rows(a, st);
    if (plan.sums) {
        int *sums = reinterpret_cast<int *>(s + plan.o_sums);
        launch_early(weight_sums_kernel, (out_dim + 7) / 8, 256, 0, st, a.w, a.w_pitch, out_dim, in_dim, sums);
        if ((rc = check_launch("weight_sums_kernel")) != NPA_OK) return rc;
        a.w_sums = sums;
    }
    return launch_int8_tcgen05(me, a, st);
}

// Memory of the two layers of an MLP, each in its turn, and of what lies between them.
struct MlpPlan {
    long long o_codes, o_scales, o_work, bytes;
    bool fused;
    MlpPlan(const void *z, long long z_pitch, const void *w1, long long w1_pitch, const void *w2, long long w2_pitch, long long rows, int in, int hidden, int out) {
        fused = mlp_int8_fused(static_cast<const float *>(z), z_pitch, w1, w1_pitch, w2, w2_pitch, rows, in, hidden, out);
        bytes = 0;
        if (fused) return;
        o_codes = round16(rows * (long long)hidden * 4);  // behind h
        o_scales = o_codes + rows * round16(hidden);
        o_work = o_scales + round16(rows * 4);
        const long long first = Int8Plan(z, NPA_FLOAT32, z_pitch, w1, w1_pitch, rows, in, hidden).bytes;
        const long long second = Int8Plan(nullptr, NPA_UINT8, round16(hidden), w2, w2_pitch, rows, hidden, out).bytes;
        bytes = o_work + (first > second ? first : second);
    }
};

int64_t npa_mlp_int8_scratch_bytes(const void *z, int64_t z_pitch, const void *w1, int64_t w1_pitch, const void *w2, int64_t w2_pitch, int64_t rows,
                                   int32_t in_dim, int32_t hidden, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || hidden <= 0 || out_dim <= 0) return 0;
    return MlpPlan(z, z_pitch, w1, w1_pitch, w2, w2_pitch, rows, in_dim, hidden, out_dim).bytes;
}

int npa_mlp_int8(const float *z, int64_t z_pitch, const void *w1, int64_t w1_pitch, const float *w1_scales, const float *b1, const void *w2, int64_t w2_pitch,
                 const float *w2_scales, float *y, int64_t rows, int32_t in_dim, int32_t hidden, int32_t out_dim, void *scratch, int64_t scratch_bytes,
                 void *stream) {
    const char *me = "npa_mlp_int8";
    int rc = check_rows(me, rows, in_dim);
    if (rc != NPA_OK) return rc;
    if (hidden <= 0 || out_dim <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: hidden and out_dim must be positive", me);
    if (!z || !w1 || !w1_scales || !b1 || !w2 || !w2_scales || !y) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be there", me);
    const MlpPlan plan(z, z_pitch, w1, w1_pitch, w2, w2_pitch, rows, in_dim, hidden, out_dim);
    if (plan.bytes && (!scratch || (uintptr_t)scratch % 16)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: scratch must be there, 16-byte aligned", me);
    if (scratch_bytes < plan.bytes)
        return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, plan.bytes);
    if (((uintptr_t)z | (uintptr_t)y | (uintptr_t)w1_scales | (uintptr_t)b1 | (uintptr_t)w2_scales) % 4)
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be aligned to its type", me);
    if (z_pitch < 0 || w1_pitch < 0 || w2_pitch < 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: pitches must not be negative", me);
    if (plan.fused)
        return launch_mlp_int8(me, z, w1, w1_pitch, w1_scales, b1, w2, w2_pitch, w2_scales, y, rows, in_dim, out_dim, (cudaStream_t)stream);
    char *p = static_cast<char *>(scratch), *codes = p + plan.o_codes, *work = p + plan.o_work;
    float *h = reinterpret_cast<float *>(p), *scales = reinterpret_cast<float *>(p + plan.o_scales);
    rc = npa_linear_int8(z, NPA_FLOAT32, z_pitch, nullptr, w1, w1_pitch, w1_scales, b1, NPA_FLOAT32, 1, h, NPA_FLOAT32, rows, in_dim, hidden, work,
                         scratch_bytes - plan.o_work, stream);
    if (rc != NPA_OK) return rc;
    rc = launch_quantize(h, NPA_FLOAT32, hidden, rows, hidden, true, codes, round16(hidden), scales, (cudaStream_t)stream);
    if (rc != NPA_OK) return rc;
    return npa_linear_int8(codes, NPA_UINT8, round16(hidden), scales, w2, w2_pitch, w2_scales, nullptr, 0, 0, y, NPA_FLOAT32, rows, hidden, out_dim, work,
                           scratch_bytes - plan.o_work, stream);
}

}  // extern "C"
