// The product of 8-bit codes on the fifth-generation tensor cores (int8.cu has the definition and the kernel for few rows).
//
//     out[m, n] = act( float(sum_k x[m, k] w[n, k]) * (s[m] * t[n]) + bias[n] )
//
// tcgen05.mma kind::i8, M = 128, K = 32 bytes an instruction, 32-bit integer accumulators in tensor memory: exact, in any order.  Both
// operands are rows with the summed index contiguous and come through TMA into 128-byte-swizzled stages of 128 bytes of K; what lies
// beyond the rows, the channels or the length is filled with zeros, which add nothing.  One persistent CTA per SM:
//
//   * one lane issues the loads of a stage (128 rows of x, BN of w), kStages ahead;
//   * one lane issues its four MMAs and hands the stage back;
//   * four warps (lane = row) turn a finished accumulator into values, 32 columns at a time through shared memory, so that rows leave in
//     whole sectors, while the MMAs of the next tile fill the other accumulator.
//
// 8,192 x 4,096 x 4,096 to bf16: 103 us, 2.67 POP/s, the tensor pipe 66 % busy.  Shared memory bounds it: an MMA of 128 x 256 x 32 reads 12 KB
// of operands that TMA wrote there once, 192 clocks at 128 bytes each, against the 128 clocks that it computes.  A tile shared by two SMs would
// halve w's part of that; not built.  The width BN of a tile follows from the number of tiles (int8_width).  Waits are bounded as in umma.cuh.
#include <mutex>

#include "int8.cuh"
#include "int8_tma.cuh"

namespace npa {

constexpr int kI8Rows = 128;                  // of a tile
constexpr int kI8WarpLoad = 0, kI8WarpMma = 1, kI8Epilogue0 = 4, kI8EpilogueWarps = 4;
constexpr int kI8Threads = (kI8Epilogue0 + kI8EpilogueWarps) * 32;
constexpr int kI8StagePitch = 32 * 4 + 16;    // bytes of a staged row of 32 values of up to 4 bytes: 16-byte stores of eight rows cover all banks

template <int BN>
struct Int8Shape {
    static constexpr int kStageBytes = (kI8Rows + BN) * kI8Chunk;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kTmemCols = 2 * BN;  // two accumulators (a power of two, at least 32)
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kI8EpilogueWarps * 32 * kI8StagePitch + 2 * 3 * BN * 4;
    static_assert(kSmem <= 226 * 1024, "shared memory of a CTA, with a kilobyte for the barriers");
};

struct Int8Shared {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], columns;
    uint32_t tmem_base;
    int abort;
};

struct Int8TileArgs {
    const float *x_scales, *w_scales;
    const int *w_sums;
    const void *bias;
    int bias_type, relu;
    void *out;
    long long rows;
    int out_dim, chunks, tiles_m, tiles_n, band, m_inner;
    unsigned *status;
};

// Tile t as (row tile, column tile): the dimension with fewer tiles runs first, in bands of `band`, so that the tiles in flight
// share their operands in L2.
__device__ __forceinline__ void int8_tile(const Int8TileArgs &a, int t, int &m, int &n) {
    const int inner = a.m_inner ? a.tiles_m : a.tiles_n, outer = a.m_inner ? a.tiles_n : a.tiles_m;
    const int per_band = a.band * outer, b = t / per_band, rest = t - b * per_band;
    const int width = min(a.band, inner - b * a.band), o = rest / width, i = b * a.band + rest - o * width;
    m = a.m_inner ? i : o;
    n = a.m_inner ? o : i;
}

template <typename T, int BN>
__global__ void __launch_bounds__(kI8Threads, 1) int8_umma_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
                                                                  const __grid_constant__ Int8TileArgs a) {
    using S = Int8Shape<BN>;
    extern __shared__ uint8_t int8_smem_raw[];
    __shared__ Int8Shared sh;
    uint8_t *base = int8_smem_raw + ((1024u - (smem_u32(int8_smem_raw) & 1023u)) & 1023u);
    uint8_t *staged = base + S::kStages * S::kStageBytes;
    float *columns = reinterpret_cast<float *>(staged + kI8EpilogueWarps * 32 * kI8StagePitch);  // [2][scale | bias | sums][BN]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    after_previous_kernel();  // before the tensor memory is asked for: the kernel before may still want it
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
        }
        for (int q = 0; q < 2; ++q) {
            mbar_init(&sh.acc_full[q], 1);
            mbar_init(&sh.acc_empty[q], kI8EpilogueWarps);
        }
        mbar_init(&sh.columns, kI8EpilogueWarps);
        sh.abort = 0;
        mbar_fence_init();
    }
    if (warp == kI8WarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(S::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = sh.tmem_base;
    const int tiles = a.tiles_m * a.tiles_n;
    bool ok = true;

    if (warp == kI8WarpLoad) {
        if (lane == 0) {
            int s = 0;
            unsigned ph = 1;
#pragma unroll 1
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                int m, n;
                int8_tile(a, t, m, n);
#pragma unroll 1
                for (int c = 0; c < a.chunks; ++c) {
                    if (!(ok = umma_wait(&sh.empty[s], ph, &sh.abort))) break;
                    mbar_arrive_expect(&sh.full[s], (unsigned)S::kStageBytes);
                    uint8_t *dst = base + s * S::kStageBytes;
                    tma_load_2d(dst, &x_map, c * kI8Chunk, m * kI8Rows, &sh.full[s]);
                    tma_load_2d(dst + kI8Rows * kI8Chunk, &w_map, c * kI8Chunk, n * BN, &sh.full[s]);
                    if (++s == S::kStages) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (!ok) {
                atomicOr(a.status, INT8_STATUS_LOAD);
                __nanosleep(20000);  // loads issued just before the flag was seen land before the CTA leaves
            }
        }
        __syncwarp();
    } else if (warp == kI8WarpMma) {
        if (lane == 0) {
            const unsigned idesc = i8_idesc(BN);
            const uint64_t desc0 = umma_desc(smem_u32(base));
            int s = 0, it = 0;
            unsigned ph = 0;
#pragma unroll 1
            for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++it) {
                const int acc = it & 1;
                if (!(ok = umma_wait(&sh.acc_empty[acc], ((it >> 1) & 1) ^ 1, &sh.abort))) break;
                tc_fence_after();
                const unsigned d = tmem + acc * BN;
#pragma unroll 1
                for (int c = 0; c < a.chunks; ++c) {
                    if (!(ok = umma_wait(&sh.full[s], ph, &sh.abort))) break;
                    tc_fence_after();
                    const uint64_t xd = desc0 + (uint64_t)((s * S::kStageBytes) >> 4), wd = xd + (uint64_t)((kI8Rows * kI8Chunk) >> 4);
#pragma unroll
                    for (int ks = 0; ks < kI8Chunk / 32; ++ks) umma_i8(d, xd + 2ull * ks, wd + 2ull * ks, idesc, (c | ks) != 0);
                    umma_commit(&sh.empty[s]);
                    if (c == a.chunks - 1) umma_commit(&sh.acc_full[acc]);
                    if (++s == S::kStages) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) break;
            }
            if (!ok) atomicOr(a.status, INT8_STATUS_MMA);
        }
        __syncwarp();
    } else if (warp >= kI8Epilogue0) {
        const int quarter = warp & 3, e = threadIdx.x - kI8Epilogue0 * 32;
        uint8_t *mine = staged + quarter * 32 * kI8StagePitch;
        const unsigned tlane = tmem + ((unsigned)(quarter * 32) << 16);
        const bool vectors = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)((long long)a.out_dim * (long long)sizeof(T))) % 16) == 0;
        int it = 0;
#pragma unroll 1
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++it) {
            int m, n;
            int8_tile(a, t, m, n);
            const int acc = it & 1, n0 = n * BN;
            const long long row0 = (long long)m * kI8Rows + quarter * 32;
            const int nrows = a.rows - row0 < 32 ? (int)(a.rows - row0) : 32;  // may be <= 0
            // the columns' scales and biases: the other half of this memory may still be read for the tile before
            float *scale = columns + acc * 3 * BN, *bias = scale + BN;
            int *sums = reinterpret_cast<int *>(bias + BN);
            for (int c = e; c < BN; c += kI8EpilogueWarps * 32) {
                const bool there = n0 + c < a.out_dim;
                scale[c] = there ? __ldg(a.w_scales + n0 + c) : 0.f;
                bias[c] = there && a.bias ? load_value(a.bias, a.bias_type, n0 + c) : 0.f;
                sums[c] = there && a.w_sums ? 128 * __ldg(a.w_sums + n0 + c) : 0;
            }
            const float row_scale = lane < nrows ? __ldg(a.x_scales + row0 + lane) : 0.f;
            // (a bounded wait as all others: at a barrier of the hardware a warp would stay for good when another has given up and left)
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.columns);
            if (!(ok = umma_wait(&sh.columns, it & 1, &sh.abort))) break;
            if (!(ok = umma_wait(&sh.acc_full[acc], (it >> 1) & 1, &sh.abort, kUmmaWaitNs, 100))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += 32) {
                unsigned r[2][16];
                tmem_ld16(tlane + acc * BN + c0, r[0]);
                tmem_ld16(tlane + acc * BN + c0 + 16, r[1]);
                tc_wait_ld();
                if (c0 + 32 >= BN) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.acc_empty[acc]);
                }
                if (n0 + c0 >= a.out_dim) continue;  // (the last block hands the accumulator back all the same)
                constexpr int kEach = 16 / sizeof(T);
#pragma unroll
                for (int q = 0; q < 32 / kEach; ++q) {
                    union {
                        uint4 quad;
                        T value[kEach];
                    } u;
#pragma unroll
                    for (int j = 0; j < kEach; ++j) {
                        const int c = q * kEach + j;
                        u.value[j] = from_float<T>(int8_value((int)r[c / 16][c % 16] + sums[c0 + c], row_scale, scale[c0 + c], a.bias != nullptr, bias[c0 + c], a.relu != 0));
                    }
                    *reinterpret_cast<uint4 *>(mine + lane * kI8StagePitch + 16 * q) = u.quad;
                }
                __syncwarp();
                T *out = static_cast<T *>(a.out) + row0 * a.out_dim + n0 + c0;
                if (vectors) {
                    constexpr int kLanes = 32 / kEach;  // of 16 bytes for a row
                    const int c = (lane % kLanes) * kEach;
                    if (n0 + c0 + c < a.out_dim) {  // (out_dim is a multiple of kEach)
#pragma unroll
                        for (int i = 0; i < kLanes; ++i) {
                            const int rr = i * (32 / kLanes) + lane / kLanes;
                            if (rr < nrows)
                                *reinterpret_cast<uint4 *>(out + (long long)rr * a.out_dim + c) =
                                    *reinterpret_cast<const uint4 *>(mine + rr * kI8StagePitch + (lane % kLanes) * 16);
                        }
                    }
                } else if (n0 + c0 + lane < a.out_dim) {
#pragma unroll 8
                    for (int rr = 0; rr < nrows; ++rr) out[(long long)rr * a.out_dim + lane] = reinterpret_cast<const T *>(mine + rr * kI8StagePitch)[lane];
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) atomicOr(a.status, INT8_STATUS_EPILOGUE);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kI8WarpMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static std::mutex mu;
    static EncodeTiled fn = nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(p);
    }
    return fn;
}

int byte_rows_map(const char *me, CUtensorMap *map, const void *p, long long pitch, long long rows, int cols, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(NPA_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", me);
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)kI8Chunk, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(NPA_ERR_CUDA, "%s: cuTensorMapEncodeTiled: error %d", me, (int)rc);
    return NPA_OK;
}

template <typename T, int BN>
static int launch_int8_shape(const char *me, const Int8Args &a, Int8TileArgs &t, cudaStream_t st) {
    using S = Int8Shape<BN>;
    CUtensorMap x_map, w_map;
    int rc = byte_rows_map(me, &x_map, a.x, a.x_pitch, a.rows, a.in, kI8Rows);
    if (rc == NPA_OK) rc = byte_rows_map(me, &w_map, a.w, a.w_pitch, a.out_dim, a.in, BN);
    if (rc != NPA_OK) return rc;
    int ctas = 0;  // also raises the kernel's limit of shared memory on this device
    rc = persistent_ctas(int8_umma_kernel<T, BN>, kI8Threads, S::kSmem, &ctas);
    if (rc != NPA_OK) return rc;
    const long long tiles_m = (a.rows + kI8Rows - 1) / kI8Rows, tiles_n = (a.out_dim + BN - 1) / BN, tiles = tiles_m * tiles_n;
    if (tiles > ((long long)1 << 30)) return fail(NPA_ERR_UNSUPPORTED, "%s: supports fewer than 2^30 tiles", me);
    t.tiles_m = (int)tiles_m;
    t.tiles_n = (int)tiles_n;
    t.m_inner = tiles_m < tiles_n;
    const int inner = t.m_inner ? t.tiles_m : t.tiles_n;
    t.band = inner < 16 ? inner : 16;
    launch_early(int8_umma_kernel<T, BN>, (int)(tiles < ctas ? tiles : ctas), kI8Threads, (size_t)S::kSmem, st, x_map, w_map, t);
    return check_launch("int8_umma_kernel");
}

// Columns of a tile: the time of a CTA is its tiles times what one of them loads, 128 + BN rows a chunk, or computes.  Measured with 32, 64,
// 128, 256, us (with the quantiser, bf16, L2 flushed): 333 x 2,048 x 5,120 33.8, 23.6, 19.5 (taken), 23.6;  1,024 cubed 17.4, 15.4 (taken),
// 17.4, 19.5;  2,048 cubed 54.3, 37.9, 29.7, 27.6 (taken);  100,000 x 128 x 35 37.9, 35.8 (taken), 37.9, 42.0.
static int int8_width(long long rows, int out_dim) {
    int best = 256;
    long long least = -1;
    for (int bn = 256; bn >= 32; bn /= 2) {
        const long long tiles = (rows + kI8Rows - 1) / kI8Rows * ((out_dim + bn - 1) / bn), cost = (tiles + 147) / 148 * (128 + bn);
        if (least < 0 || cost < least) {
            least = cost;
            best = bn;
        }
    }
    return best;
}

template <typename T>
static int launch_int8_type(const char *me, const Int8Args &a, Int8TileArgs &t, cudaStream_t st) {
    switch (int8_width(a.rows, a.out_dim)) {
        case 256: return launch_int8_shape<T, 256>(me, a, t, st);
        case 128: return launch_int8_shape<T, 128>(me, a, t, st);
        case 64: return launch_int8_shape<T, 64>(me, a, t, st);
        default: return launch_int8_shape<T, 32>(me, a, t, st);
    }
}

int launch_int8_tcgen05(const char *me, const Int8Args &a, cudaStream_t st) {
    Int8TileArgs t = {};
    t.x_scales = a.x_scales; t.w_scales = a.w_scales; t.w_sums = a.w_sums; t.bias = a.bias; t.bias_type = a.bias_type; t.relu = a.relu; t.out = a.out;
    t.rows = a.rows; t.out_dim = a.out_dim; t.chunks = (a.in + kI8Chunk - 1) / kI8Chunk;
    if (!(t.status = umma_status_word())) return fail(NPA_ERR_CUDA, "%s: no status word", me);
    if (a.out_type == NPA_FLOAT32) return launch_int8_type<float>(me, a, t, st);
    if (a.out_type == NPA_FLOAT16) return launch_int8_type<__half>(me, a, t, st);
    return launch_int8_type<__nv_bfloat16>(me, a, t, st);
}

}  // namespace npa
