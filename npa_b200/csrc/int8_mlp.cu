// Both layers of the adaptation MLP in 8-bit integers, in one kernel (hidden width 128; int8.cu has the definitions):
//
//     q, s = codes of z's rows;  h = relu(float(q w1^T) * (s t1) + b1);  p, u = unsigned codes of h's rows;  y = float(p w2^T) * (u t2)
//
// Memory gives the time: z is read once (4 bytes an input) and y written once.  Between them a row exists as codes in shared memory and
// sums in tensor memory only; the two products are 10 MMAs of kind::i8 for 128 rows at 163 inputs.  What is left to arrange is the
// arithmetic around them, some 7 instructions a value of z and 12 of h:
//
//   * one lane brings z in slots of 32 rows (contiguous blocks, bulk copies), kSlots ahead;
//   * eight warps make codes: eight rows at a time, lane = column, so that their maxima share shuffles;
//   * one lane issues the MMAs; w1 and w2 come once per CTA through TMA and stay;
//   * eight warps, two for a quarter of the rows, turn sums into h (64 units a thread, kept in registers between the maximum and the
//     codes) and the second layer's sums into rows of y, which leave as one contiguous block.
//
// Measured (B200, us): 80 for 262,144 rows of 163 and 35 (the bytes alone: 32), 9.5 for 2,500 rows of 66 and 18.  Nothing is full: 20,500
// instructions a tile of 128 rows take 46 % of the issue slots, DRAM moves 2 TB/s, the tensor pipe is 4 % busy.  What is left is order: at more than
// 128 inputs there is room for one buffer of codes, so that the converters wait for each tile's first product, and h, its maximum, the
// partner's half, the codes and y of the tile before are one chain in the epilogue.
//
// The MMA is given signed codes on both sides (i8_idesc; it would take either side unsigned): h's are shifted by 128, and 128 times the sum of
// w2's row comes back in the epilogue.
// Waits are bounded as in umma.cuh.
#include "int8.cuh"
#include "int8_tma.cuh"

namespace npa {

constexpr int kMlpRows = 128, kMlpHidden = 128, kMlpMaxIn = 256, kMlpMaxOut = 64;
constexpr int kMlpSlotRows = 32, kMlpMaxSlots = 8;
constexpr int kMlpConverters = 8, kMlpEpilogue = 8, kMlpWarpMma = 16, kMlpWarpCopy = 17, kMlpThreads = 18 * 32;
constexpr int kMlpTile = kMlpRows * 128;  // bytes of 128 rows of 128 codes
constexpr int kMlpAcc = 128, kMlpYCol = 256;

struct MlpInt8Shared {
    uint64_t weights, raw_full[kMlpMaxSlots], raw_empty[kMlpMaxSlots], z_full[2], z_empty[2], acc_full[2], acc_empty[2], h_ready[2], h_empty[2], y_full[2],
        y_written, y_copied, pair[4];
    alignas(16) float t1[kMlpHidden], b1[kMlpHidden], t2[kMlpMaxOut];
    alignas(16) int sums[kMlpMaxOut];
    float scale[4][kMlpRows];               // of z's rows, four tiles
    unsigned largest[2][kMlpEpilogue][32];  // of h's halves
    float u[4][kMlpRows];                   // scales of h's rows
    uint32_t tmem_base;
    int abort;
};

struct MlpInt8Args {
    const float *z;
    const int8_t *w2;
    long long w2_pitch;
    const float *t1, *b1, *t2;
    float *y;
    long long rows;
    int in, out, chunks, zbufs, slots, slot_bytes, n2, tiles, blocks;  // blocks: of 32 columns of z
    unsigned *status;
};

// Byte of code (row, k), k < 128, in a swizzled tile.
__device__ __forceinline__ int code_place(int row, int k) { return row * 128 + ((((k >> 4) ^ row) & 7) << 4) + (k & 15); }

// Codes of eight rows of `in` <= 32 kBlocks values that follow one another at p; `codes`: the first of them in a swizzled tile, `scales`
// its scale.  A lane works out the scale of one row (four lanes the same) and hands it round.
template <int kBlocks>
__device__ __forceinline__ void convert_rows(const float *p, int in, uint8_t *codes, float *scales, int lane) {
    float v[8][kBlocks], largest[8];
    const bool last = 32 * (kBlocks - 1) + lane < in;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const float *row = p + r * in + lane;
        largest[r] = 0.f;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            v[r][b] = b + 1 < kBlocks || last ? row[32 * b] : 0.f;
            largest[r] = larger(largest[r], fabsf(v[r][b]));
        }
    }
    float inverse;
    const float scale = row_scale(magnitude(gather_max8(largest)), 127.f, inverse);
    if (lane % 4 == 0) scales[lane / 4] = scale;
    // place of (row r, column 32 b + lane): units of 16 codes change places by the row's lowest three bits, the lane's half by the first
    const int place[2] = {((lane >> 4) << 4) + (lane & 15), (((lane >> 4) ^ 1) << 4) + (lane & 15)};
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const float s = __shfl_sync(kFull, scale, 4 * r), i = __shfl_sync(kFull, inverse, 4 * r);
        unsigned code[kBlocks];
        row_codes<kBlocks, true>(v[r], s, i, code);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) codes[(b / 4) * kMlpTile + r * 128 + (((2 * (b % 4)) ^ (r & 6)) << 4) + place[r & 1]] = (uint8_t)code[b];
    }
}

template <int kBlocks>
__global__ void __launch_bounds__(kMlpThreads, 1) mlp_int8_kernel(const __grid_constant__ CUtensorMap w1_map, const __grid_constant__ CUtensorMap w2_map,
                                                                  const __grid_constant__ MlpInt8Args a) {
    after_previous_kernel();
    extern __shared__ uint8_t mlp8_raw[];
    __shared__ MlpInt8Shared sh;
    uint8_t *base = mlp8_raw + ((1024u - (smem_u32(mlp8_raw) & 1023u)) & 1023u);
    uint8_t *w1 = base, *w2 = w1 + a.chunks * kMlpTile, *zc = w2 + a.n2 * 128, *hc = zc + a.zbufs * a.chunks * kMlpTile, *raw = hc + 2 * kMlpTile;
    float *ytile = reinterpret_cast<float *>(raw + a.slots * a.slot_bytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&sh.weights, 1);
        for (int s = 0; s < a.slots; ++s) {
            mbar_init(&sh.raw_full[s], 1);
            mbar_init(&sh.raw_empty[s], 4);
        }
        for (int q = 0; q < 2; ++q) {
            mbar_init(&sh.z_full[q], 16);  // four warps for each of four slots
            mbar_init(&sh.z_empty[q], 1);
            mbar_init(&sh.acc_full[q], 2);  // the products, and the MMA lane itself: what it has seen of the scales the epilogue sees
            mbar_init(&sh.acc_empty[q], kMlpEpilogue);
            mbar_init(&sh.h_ready[q], kMlpEpilogue);
            mbar_init(&sh.h_empty[q], 1);
            mbar_init(&sh.y_full[q], 2);
        }
        mbar_init(&sh.y_written, kMlpEpilogue);
        mbar_init(&sh.y_copied, kMlpEpilogue);
        for (int q = 0; q < 4; ++q) mbar_init(&sh.pair[q], 2);
        sh.abort = 0;
        mbar_fence_init();
    }
    for (int c = threadIdx.x; c < kMlpHidden; c += kMlpThreads) {
        sh.t1[c] = __ldg(a.t1 + c);
        sh.b1[c] = __ldg(a.b1 + c);
    }
    if (threadIdx.x < kMlpMaxOut) sh.t2[threadIdx.x] = threadIdx.x < a.out ? __ldg(a.t2 + threadIdx.x) : 0.f;
    for (int n = warp; n < kMlpMaxOut; n += kMlpThreads / 32) {
        int sum = 0;
        if (n < a.out) sum = __dp4a(__ldg(reinterpret_cast<const int *>(a.w2 + n * a.w2_pitch) + lane), 0x01010101, 0);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(kFull, sum, d);
        if (lane == 0) sh.sums[n] = 128 * sum;
    }
    if (warp == kMlpWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = sh.tmem_base;
    const int ntile = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    auto row_of = [&](int it) { return ((long long)blockIdx.x + (long long)it * gridDim.x) * kMlpRows; };
    // a slot whose 32 rows all exist comes by bulk copy; what is left of the last one is read by the warps that need it
    auto whole = [&](long long row0) { return row0 + kMlpSlotRows <= a.rows; };
    bool ok = true;

    if (warp == kMlpWarpCopy) {
        if (lane == 0) {
            mbar_arrive_expect(&sh.weights, (unsigned)(a.chunks * kMlpTile + a.n2 * 128));
            for (int c = 0; c < a.chunks; ++c) tma_load_2d(w1 + c * kMlpTile, &w1_map, c * kI8Chunk, 0, &sh.weights);
            tma_load_2d(w2, &w2_map, 0, 0, &sh.weights);
            int s = 0;
            unsigned ph = 1;
#pragma unroll 1
            for (int q = 0; q < 4 * ntile && ok; ++q) {
                const long long row0 = row_of(q >> 2) + (q & 3) * kMlpSlotRows;
                if (!(ok = umma_wait(&sh.raw_empty[s], ph, &sh.abort))) break;
                if (whole(row0)) {
                    mbar_arrive_expect(&sh.raw_full[s], (unsigned)a.slot_bytes);
                    bulk_copy_g2s(raw + s * a.slot_bytes, a.z + row0 * a.in, (unsigned)a.slot_bytes, &sh.raw_full[s]);
                } else {
                    mbar_arrive(&sh.raw_full[s]);
                }
                if (++s == a.slots) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!ok) {
                atomicOr(a.status, INT8_STATUS_LOAD);
                __nanosleep(20000);  // copies in flight land before the CTA leaves
            }
        }
        __syncwarp();
    } else if (warp == kMlpWarpMma) {
        if (lane == 0) {
            const unsigned id1 = i8_idesc(128), id2 = i8_idesc(a.n2);
            const uint64_t w1d = umma_desc(smem_u32(w1)), w2d = umma_desc(smem_u32(w2));
            const int steps = (a.in + 31) / 32;
            ok = umma_wait(&sh.weights, 0, &sh.abort);
            auto second = [&](int t) -> bool {
                const int b = t & 1;
                if (!umma_wait(&sh.h_ready[b], (t >> 1) & 1, &sh.abort)) return false;
                tc_fence_after();
                const uint64_t hd = umma_desc(smem_u32(hc + b * kMlpTile));
                for (int ks = 0; ks < 4; ++ks) umma_i8(tmem + kMlpYCol + b * 64, hd + 2 * ks, w2d + 2 * ks, id2, ks != 0);
                umma_commit(&sh.h_empty[b]);
                umma_commit(&sh.y_full[b]);
                mbar_arrive(&sh.y_full[b]);
                return true;
            };
            int zb = 0;
            unsigned zph = 0;
#pragma unroll 1
            for (int t = 0; t < ntile && ok; ++t) {
                const int b = t & 1;
                if (!(ok = umma_wait(&sh.z_full[zb], zph, &sh.abort))) break;
                if (!(ok = umma_wait(&sh.acc_empty[b], ((t >> 1) & 1) ^ 1, &sh.abort))) break;
                tc_fence_after();
                const uint64_t zd = umma_desc(smem_u32(zc + zb * a.chunks * kMlpTile));
                for (int ks = 0; ks < steps; ++ks) {
                    const uint64_t o = (uint64_t)((ks >> 2) * (kMlpTile >> 4) + 2 * (ks & 3));
                    umma_i8(tmem + b * kMlpAcc, zd + o, w1d + o, id1, ks != 0);
                }
                umma_commit(&sh.z_empty[zb]);
                umma_commit(&sh.acc_full[b]);
                mbar_arrive(&sh.acc_full[b]);
                if (++zb == a.zbufs) {
                    zb = 0;
                    zph ^= 1;
                }
                if (t > 0) ok = second(t - 1);
            }
            if (ok && ntile > 0) ok = second(ntile - 1);
            if (!ok) {
                atomicOr(a.status, INT8_STATUS_MMA);
                __nanosleep(20000);
            }
        }
        __syncwarp();
    } else if (warp < kMlpConverters) {
        // warps 0 to 3 take the even slots, 4 to 7 the odd ones, eight rows each
        const int group = warp >> 2, mine = (warp & 3) * 8;
        int zb = 0;
        unsigned zph = 1;
#pragma unroll 1
        for (int t = 0; t < ntile && ok; ++t) {
            if (!(ok = umma_wait(&sh.z_empty[zb], zph, &sh.abort))) break;
            uint8_t *codes = zc + zb * a.chunks * kMlpTile;
#pragma unroll 1
            for (int part = group; part < 4; part += 2) {
                const int q = 4 * t + part, s = q % a.slots;
                if (!(ok = umma_wait(&sh.raw_full[s], (q / a.slots) & 1, &sh.abort))) break;
                const long long row0 = row_of(t) + part * kMlpSlotRows;
                const int first = part * kMlpSlotRows + mine;
                float *p = reinterpret_cast<float *>(raw + s * a.slot_bytes) + mine * a.in;
                if (!whole(row0)) {  // this warp's rows of the last slot, as far as they exist
                    const long long from = (row0 + mine) * a.in, end = a.rows * a.in;
                    for (int k = lane; k < 8 * a.in; k += 32) p[k] = from + k < end ? __ldg(a.z + from + k) : 0.f;
                    __syncwarp();
                }
                convert_rows<kBlocks>(p, a.in, codes + first * 128, &sh.scale[t & 3][first], lane);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sh.z_full[zb]);
                    mbar_arrive(&sh.raw_empty[s]);
                }
            }
            if (++zb == a.zbufs) {
                zb = 0;
                zph ^= 1;
            }
        }
        if (!ok && lane == 0) atomicOr(a.status, INT8_STATUS_LOAD);
    } else {
        const int e = warp - kMlpConverters, quarter = warp & 3, half = e >> 2, row = quarter * 32 + lane;
        const unsigned tlane = tmem + ((unsigned)(quarter * 32) << 16);
        auto leave = [&](int t) -> bool {  // y of tile t
            const int b = t & 1;
            const long long row0 = row_of(t);
            if (!umma_wait(&sh.y_copied, (t & 1) ^ 1, &sh.abort)) return false;
            if (!umma_wait(&sh.y_full[b], (t >> 1) & 1, &sh.abort)) return false;
            tc_fence_after();
            const float u = sh.u[t & 3][row];
#pragma unroll 1
            for (int c0 = 16 * half; c0 < a.n2; c0 += 32) {
                unsigned r[16];
                tmem_ld16(tlane + kMlpYCol + 64 * b + c0, r);
                tc_wait_ld();
                float y[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = __fmul_rn(__int2float_rn((int)r[j] + sh.sums[c0 + j]), __fmul_rn(u, sh.t2[c0 + j]));
                put_16(ytile + row * a.out + c0, a.out - c0, a.out, lane, y);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.y_written);
            if (!umma_wait(&sh.y_written, t & 1, &sh.abort)) return false;
            const int here = a.rows - row0 < kMlpRows ? (int)(a.rows - row0) : kMlpRows, total = here * a.out;
            float *out = a.y + row0 * a.out;  // (128 rows of any width are a multiple of 16 bytes)
            const int at = e * 32 + lane;
            const int quads = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 ? total / 4 : 0;
            for (int q = at; q < quads; q += kMlpEpilogue * 32) reinterpret_cast<float4 *>(out)[q] = reinterpret_cast<const float4 *>(ytile)[q];
            for (int q = 4 * quads + at; q < total; q += kMlpEpilogue * 32) out[q] = ytile[q];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.y_copied);
            return true;
        };
#pragma unroll 1
        for (int t = 0; t < ntile; ++t) {
            const int b = t & 1;
            if (!(ok = umma_wait(&sh.acc_full[b], (t >> 1) & 1, &sh.abort))) break;
            tc_fence_after();
            const float s = sh.scale[t & 3][row];
            float v[4][16];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int c0 = 64 * half + 16 * c;
                unsigned r[16];
                tmem_ld16(tlane + b * kMlpAcc + c0, r);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 t1 = *reinterpret_cast<const float4 *>(&sh.t1[c0 + j]), b1 = *reinterpret_cast<const float4 *>(&sh.b1[c0 + j]);
                    const float tw[4] = {t1.x, t1.y, t1.z, t1.w}, bw[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // (sums of 256 products of 127 x 127 are below 2^22: added to 1.5 * 2^23 in its last bits, they become numbers)
                        const float sum = __int_as_float((int)r[j + i] + __float_as_int(kRoundWhole)) - kRoundWhole;
                        v[c][j + i] = larger(__fadd_rn(__fmul_rn(sum, __fmul_rn(s, tw[i])), bw[i]), 0.f);
                        most = larger(most, v[c][j + i]);
                    }
                }
            }
            tc_fence_before();
            unsigned largest = magnitude(most);
            sh.largest[b][e][lane] = largest;
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.acc_empty[b]);
                mbar_arrive(&sh.pair[quarter]);
            }
            if (!(ok = umma_wait(&sh.pair[quarter], t & 1, &sh.abort))) break;
            largest = max(largest, sh.largest[b][e ^ 4][lane]);
            float inverse;
            const float u = row_scale(largest, 255.f, inverse);
            if (half == 0) sh.u[t & 3][row] = u;  // (read by both halves behind the next barrier of the tile)
            if (!(ok = umma_wait(&sh.h_empty[b], ((t >> 1) & 1) ^ 1, &sh.abort))) break;
            uint8_t *to = hc + b * kMlpTile;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                unsigned code[16], w[4];
                row_codes<16, true>(v[c], u, inverse, code);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack_codes(code[4 * j], code[4 * j + 1], code[4 * j + 2], code[4 * j + 3]) ^ 0x80808080u;
                *reinterpret_cast<uint4 *>(to + code_place(row, 64 * half + 16 * c)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.h_ready[b]);
            if (t > 0 && !(ok = leave(t - 1))) break;
        }
        if (ok && ntile > 0) ok = leave(ntile - 1);
        if (!ok && lane == 0) atomicOr(a.status, INT8_STATUS_EPILOGUE);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMlpWarpMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
bool mlp_int8_fused(const float *z, long long z_pitch, const void *w1, long long w1_pitch, const void *w2, long long w2_pitch, long long rows, int in,
                    int hidden, int out) {
    return hidden == kMlpHidden && in <= kMlpMaxIn && out <= kMlpMaxOut && (z_pitch == in || rows == 1) &&
           ((uintptr_t)z | (uintptr_t)w1 | (uintptr_t)w1_pitch | (uintptr_t)w2 | (uintptr_t)w2_pitch) % 16 == 0 && w1_pitch >= in && w2_pitch >= hidden;
}

template <int kBlocks>
static int launch_mlp_int8_shape(const CUtensorMap &w1_map, const CUtensorMap &w2_map, const MlpInt8Args &a, int smem, cudaStream_t st) {
    int ctas = 0;
    const int rc = persistent_ctas(mlp_int8_kernel<kBlocks>, kMlpThreads, (size_t)smem, &ctas);
    if (rc != NPA_OK) return rc;
    launch_early(mlp_int8_kernel<kBlocks>, a.tiles < ctas ? a.tiles : ctas, kMlpThreads, (size_t)smem, st, w1_map, w2_map, a);
    return check_launch("mlp_int8_kernel");
}

int launch_mlp_int8(const char *me, const float *z, const void *w1, long long w1_pitch, const float *t1, const float *b1, const void *w2, long long w2_pitch,
                    const float *t2, float *y, long long rows, int in, int out, cudaStream_t st) {
    MlpInt8Args a = {};
    a.z = z; a.w2 = static_cast<const int8_t *>(w2); a.w2_pitch = w2_pitch; a.t1 = t1; a.b1 = b1; a.t2 = t2; a.y = y; a.rows = rows; a.in = in; a.out = out;
    a.chunks = (in + 127) / 128;
    a.zbufs = a.chunks == 1 ? 2 : 1;
    a.slot_bytes = kMlpSlotRows * in * 4;
    a.n2 = (out + 15) / 16 * 16;
    a.tiles = (int)((rows + kMlpRows - 1) / kMlpRows);
    a.blocks = (in + 31) / 32;
    const int fixed = 1024 + a.chunks * kMlpTile + a.n2 * 128 + a.zbufs * a.chunks * kMlpTile + 2 * kMlpTile + kMlpRows * out * 4 + 16;
    const int room = 232448 - (int)sizeof(MlpInt8Shared) - 1024 - fixed;
    // an even number of them: a slot then always serves the same four warps, which see each of its phases (a wait tells two apart, no more)
    a.slots = (room / a.slot_bytes < kMlpMaxSlots ? room / a.slot_bytes : kMlpMaxSlots) & ~1;
    if (a.slots < 2) return fail(NPA_ERR_UNSUPPORTED, "%s: no room for two slots of rows", me);
    if (!(a.status = umma_status_word())) return fail(NPA_ERR_CUDA, "%s: no status word", me);
    CUtensorMap w1_map, w2_map;
    int rc = byte_rows_map(me, &w1_map, w1, w1_pitch, kMlpHidden, in, kMlpHidden);
    if (rc == NPA_OK) rc = byte_rows_map(me, &w2_map, w2, w2_pitch, out, kMlpHidden, a.n2);
    if (rc != NPA_OK) return rc;
    const int smem = fixed + a.slots * a.slot_bytes;
    switch (a.blocks) {
        case 1: return launch_mlp_int8_shape<1>(w1_map, w2_map, a, smem, st);
        case 2: return launch_mlp_int8_shape<2>(w1_map, w2_map, a, smem, st);
        case 3: return launch_mlp_int8_shape<3>(w1_map, w2_map, a, smem, st);
        case 4: return launch_mlp_int8_shape<4>(w1_map, w2_map, a, smem, st);
        case 5: return launch_mlp_int8_shape<5>(w1_map, w2_map, a, smem, st);
        case 6: return launch_mlp_int8_shape<6>(w1_map, w2_map, a, smem, st);
        case 7: return launch_mlp_int8_shape<7>(w1_map, w2_map, a, smem, st);
        default: return launch_mlp_int8_shape<8>(w1_map, w2_map, a, smem, st);
    }
}

}  // namespace npa
