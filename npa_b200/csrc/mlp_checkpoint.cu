// The adaptation MLP (hidden width 128) with an 8-bit checkpoint of its input (rows8.cuh):
//
//     y = relu(z W1^T + b1) W2^T, keeping codes(z) and the bits of the ReLU                   (mlp_checkpoint_forward_kernel)
//     zh = restore(codes),  dh = bits * (dy W2),  h = bits * (zh W1^T + b1)
//     dz = dh W1                                                                            (mlp_checkpoint_dz_kernel)
//     dW1 = dh^T zh,  db1 = sum of dh,  dW2 = dy^T h                                          (mlp_checkpoint_weights_kernel)
//
// dz and db1 are those of a backward in 32 bits, because the bits are those of the forward; dW1 and dW2 see the rounding of z to codes.
//
// All products run on the fifth-generation tensor cores at 32-bit accuracy with half the work of TF32: kind::f16 runs at twice its rate.
// A number is taken apart into a head and a tail of float16, 22 bits (the dropped tail x tail is 2^-22); zh needs no tail, its codes
// have 8 bits.  The price is float16's range, paid in powers of two, all exact:
//
//   * weights in units of their matrix, and of a row or column that lies apart from it (CkHeader): input columns, hidden units and outputs of
//     any size keep their own accuracy.  A unit of a summed index goes to the other operand or comes back into the image once in front of the
//     tiles; one of an index that stays comes back in the epilogue.  Weights that lie together take neither way;
//   * z in the forward, and dy for dz, in units of their row: rows of any size keep their accuracy, and the unit comes back in the epilogue;
//   * dy and zh for the sums over rows in the unit of the largest of their tile of 128 rows, which comes in when the tile's sum leaves the
//     accumulator, and, where they lie apart, of their column and group of columns (ck_settle);
//   * h in a unit that its products and the largest bias cannot exceed, dh times a power of two that brings its largest sum back in range.
//
// The largest of a unit is an operand of 2^14 to 2^15 (accumulators have 32 bits, only operands are short), which leaves 22 bits to what is
// up to 2^17 below it, and 2^-39 of the largest to the rest.  Nothing here can overflow.  What is not finite has no part in a unit, so that
// its neighbours keep theirs.
//
// What goes through memory is z, y, the checkpoint, dy and dz: no kernel writes a hidden layer (dh is made twice: 18 of 86 and of 127
// thousand products a row at 163 inputs and 35 outputs, against 512 bytes each way).  An addition on the tensor cores cuts off what lies
// below the sum's last bit, so products with tails come first or have a sum of their own.
//
// The layouts use that a swizzled tile of 16-bit numbers serves both ways: rows of 64 numbers (128 bytes, 128-byte swizzle) are a
// K-major operand for sums over the columns and an MN-major one for sums over the rows.  So one image of W1 ([hidden][in]) is B of
// z W1^T, A of zh W1^T and B of dh W1, and one tile of zh is B of both of its products, as is dy's.
//
// Memory is the floor (B200, 262,144 rows of 163 and 35: 512 MB, 78 us) and not what bounds them: it is the way of a tile through
// conversion, product, mask, product, one after another in what tensor and shared memory are left.  Measured there, us, each from a cold L2:
// image 6, forward 143 (the 32-bit forward that leaves its hidden layer: 143), dz 88, weights 147, their sum over CTAs 5; the parts of a
// tile's way stand at the kernels.  At 32,768 rows of 66 and 18: 6, 18, 14, 21 and 5, and the host takes 90 us a pass, 57 of them torch's engine for
// the backward.
//
// Waits are bounded as in umma.cuh; they report through npa_linear_tcgen05_status (bits 1024, 2048, 4096: MMA lane, producers, epilogue).
#include <mutex>
#include <type_traits>

#include "mlp_grad_reduce.cuh"
#include "rows8.cuh"
#include "umma.cuh"

namespace npa {

constexpr int kCkRows = 128;
constexpr int kCkTile = kCkRows * 128;   // bytes of 128 rows of 64 numbers
constexpr int kCkThreads = 12 * 32, kCkProducer0 = 8, kCkProducers = 4;  // (twelve warps: 168 registers a thread; a thirteenth would cost 40 of them)
constexpr int kCkMaxIn = 176, kCkMaxOut = 48;
constexpr int kCkHeader = 1024;          // bytes of the image in front of the matrices
constexpr int kCkRowRing = 8;            // tiles whose rows' units are kept

enum { CK_STATUS_MMA = 1024, CK_STATUS_PRODUCER = 2048, CK_STATUS_EPILOGUE = 4096 };

unsigned *umma_status_word();  // mlp_tcgen05.cu
int launch_grad_reduce(const GradReduce &a, cudaStream_t st);  // mlp_grad_tcgen05.cu

// ---- numbers ---------------------------------------------------------------------------------------------------------
// Exponent of the power of two at or below a finite magnitude; 0 for zero.
__device__ __forceinline__ int binade(unsigned magnitude_bits) { return magnitude_bits == 0 ? 0 : max((int)(magnitude_bits >> 23), 1) - 127; }
// A magnitude as a unit sees it: what is not finite has no part in it, so that its neighbours keep their accuracy.
__device__ __forceinline__ unsigned finite_magnitude(float v) {
    const unsigned m = magnitude(v);
    return m < 0x7f800000u ? m : 0u;
}
__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.f : __uint_as_float((unsigned)(min(e, 127) + 127) << 23); }
// a in the lower half.
__device__ __forceinline__ unsigned pack_halves(float a, float b) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float2 unpack_halves(unsigned v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
// The largest of what shares a unit becomes an operand of 2^kOperand to twice that, the last binade that float16 rounds without overflow:
// a tail's last bit is 2^-24, so that the top 17 binades keep 22 bits, and what lies below is off by 2^-39 of the largest.
constexpr int kOperand = 14;
// Heads and tails of two numbers.
__device__ __forceinline__ void split_halves(float a, float b, unsigned &head, unsigned &tail) {
    head = pack_halves(a, b);
    const float2 h = unpack_halves(head);
    tail = pack_halves(a - h.x, b - h.y);
}
// Byte of number (row, k), k < 64, in a swizzled tile.
__host__ __device__ constexpr int half_place(int row, int k) { return row * 128 + ((((k >> 3) ^ row) & 7) << 4) + (k & 7) * 2; }

// v 2^e, for exponents of up to twice a number's.
__device__ __forceinline__ float times_power(float v, int e) {
    const int part = max(min(e, 127), -126);
    return v * power_of_two(part) * power_of_two(max(min(e - part, 127), -126));
}

// ---- the weights' image ------------------------------------------------------------------------------------------------
// W1 in units of 2^(w1 + hidden1[j] + inputs[k]), W2 in units of 2^(w2 + hidden2[j] + outputs[c]): a channel whose largest number lies 2^kApart
// or more below the matrix's has a unit of its own, so that it is held as accurately as the largest.  Channels have 0 where that is not so.
// A hidden unit's row of W1 counts together with its bias, which is then no larger than the matrix either.
constexpr int kApart = 6, kFarthest = 100;
enum { CK_INPUTS = 1, CK_HIDDEN = 2, CK_OUTPUTS = 4 };
struct CkHeader {
    int w1, w2, b1;      // exponents of the matrices' units, and of the largest positive bias over its row's unit (-1000: there is none)
    int hidden;          // the largest hidden1[j] + hidden2[j]
    int apart;           // which of them differ (CK_HIDDEN: in the sum of both)
    int8_t hidden1[128], hidden2[128], inputs[192], outputs[64];
};
static_assert(sizeof(CkHeader) <= kCkHeader, "in front of the matrices");
struct CkImageArgs {
    const float *W1, *b1, *W2;
    long long s1o, s1i, s2o, s2i;
    int in, out, chunks;
    uint8_t *image;  // header | W1 heads [chunks] | W1 tails [chunks] | W2 heads | W2 tails, each 128 rows of 64 numbers
};
// Exponent of a channel's unit, from its largest magnitude and the matrix's exponent.
__device__ __forceinline__ int channel_unit(unsigned largest, int e) {
    const int d = binade(largest) - e;
    return largest == 0 || d > -kApart ? 0 : max(d, -kFarthest);
}
constexpr int kImageThreads = 512;
static int ck_image_blocks(int chunks) { return (chunks + 1) * 128 * 32 / kImageThreads; }  // a thread makes one pair
__global__ void __launch_bounds__(kImageThreads) mlp_checkpoint_image_kernel(const __grid_constant__ CkImageArgs a) {
    after_previous_kernel();
    __shared__ unsigned most[3], rows1[128], columns1[192], rows2[64], columns2[128];
    __shared__ int hidden1[128], inputs[192], hidden2[128], outputs[64], hidden[2];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (t < 3) most[t] = 0;
    if (t < 192) columns1[t] = 0;
    if (t < 64) rows2[t] = 0;
    if (t < 128) columns2[t] = 0;
    if (t < 2) hidden[t] = -1000;
    // this thread's pair of numbers, and, as every block looks at all weights (they are few, and a launch in between would cost more), eight
    // rows of W1 a warp and a quarter of a column of W2 a thread: loads of a fixed number, so that all are in flight at once
    const int q = blockIdx.x * kImageThreads + t, pairs1 = a.chunks * 128 * 32;
    const bool first = q < pairs1;
    const int at = first ? q : q - pairs1, row = (at >> 5) & 127, chunk = at >> 12, k0 = chunk * 64 + 2 * (at & 31);
    float v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        v[i] = first ? (k0 + i < a.in ? __ldg(a.W1 + row * a.s1o + (k0 + i) * a.s1i) : 0.f) : (k0 + i < a.out ? __ldg(a.W2 + (k0 + i) * a.s2o + row * a.s2i) : 0.f);
    constexpr int kRows1 = 8, kColumns1 = (kCkMaxIn + 31) / 32, kRows2 = 128 * kCkMaxOut / kImageThreads;
    float v1[kRows1][kColumns1], v2[kRows2];
#pragma unroll
    for (int r = 0; r < kRows1; ++r)
#pragma unroll
        for (int i = 0; i < kColumns1; ++i) {
            const int k = lane + 32 * i;
            v1[r][i] = k < a.in ? __ldg(a.W1 + (warp + 16 * r) * a.s1o + k * a.s1i) : 0.f;
        }
    const int unit2 = t & 127, c0 = t >> 7;
#pragma unroll
    for (int i = 0; i < kRows2; ++i) v2[i] = c0 + 4 * i < a.out ? __ldg(a.W2 + (c0 + 4 * i) * a.s2o + unit2 * a.s2i) : 0.f;
    const float bias = t < 128 ? __ldg(a.b1 + t) : 0.f;
    __syncthreads();
    // the largest of rows and columns, the columns as they are: that is what they are in units of their rows unless those lie apart
    // (first of everything; where that is not finite, of what is)
    auto look = [&](auto size) {
        unsigned m1[kRows1], m2[16], column[kColumns1] = {}, column2 = 0;
#pragma unroll
        for (int r = 0; r < kRows1; ++r) {
            m1[r] = 0;
#pragma unroll
            for (int i = 0; i < kColumns1; ++i) {
                const unsigned m = size(v1[r][i]);
                m1[r] = max(m1[r], m);
                column[i] = max(column[i], m);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            m2[i] = i < kRows2 ? size(v2[i]) : 0u;
            column2 = max(column2, m2[i]);
        }
        const unsigned one = gather_max8(m1), two = gather_max8(*reinterpret_cast<unsigned(*)[8]>(m2)), three = gather_max8(*reinterpret_cast<unsigned(*)[8]>(m2 + 8));
        if (lane % 4 == 0) {
            rows1[warp + 16 * (lane / 4)] = one;
            atomicMax(&rows2[c0 + 4 * (lane / 4)], two);
            if (lane < 16) atomicMax(&rows2[c0 + 4 * (8 + lane / 4)], three);
        }
        const unsigned all1 = warp_max(one), all2 = warp_max(max(two, three));
        if (lane == 0) {
            atomicMax(&most[0], all1);
            atomicMax(&most[1], all2);
        }
#pragma unroll
        for (int i = 0; i < kColumns1; ++i) atomicMax(&columns1[lane + 32 * i], column[i]);
        atomicMax(&columns2[unit2], column2);
        __syncthreads();
    };
    look([](float v) { return magnitude(v); });
    if (max(most[0], most[1]) >= 0x7f800000u) {
        __syncthreads();
        if (t < 2) most[t] = 0;
        if (t < 192) columns1[t] = 0;
        if (t < 64) rows2[t] = 0;
        if (t < 128) columns2[t] = 0;
        __syncthreads();
        look([](float v) { return finite_magnitude(v); });
    }
    const int e1 = binade(most[0]), e2 = binade(most[1]);
    int apart1 = 0, apart2 = 0;
    if (t < 128) {
        apart1 = hidden1[t] = channel_unit(max(rows1[t], min(finite_magnitude(bias), (unsigned)(e1 + 127) << 23)), e1);
        const unsigned m = warp_max(bias > 0.f ? finite_magnitude(bias * power_of_two(-apart1)) : 0u);
        if (lane == 0) atomicMax(&most[2], m);
    } else if (t < 192) {
        apart2 = outputs[t - 128] = channel_unit(rows2[t - 128], e2);
    }
    const int outputs_apart = __syncthreads_or(apart2);
    if (__syncthreads_or(apart1)) {
        if (t < 192) columns1[t] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kColumns1; ++i) {
            unsigned m = 0;
#pragma unroll
            for (int r = 0; r < kRows1; ++r) m = max(m, finite_magnitude(v1[r][i] * power_of_two(-hidden1[warp + 16 * r])));
            atomicMax(&columns1[lane + 32 * i], m);
        }
        __syncthreads();
    }
    if (outputs_apart) {
        if (t < 128) columns2[t] = 0;
        __syncthreads();
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < kRows2; ++i) m = max(m, finite_magnitude(v2[i] * power_of_two(-outputs[c0 + 4 * i])));
        atomicMax(&columns2[unit2], m);
        __syncthreads();
    }
    int apart = 0;
    if (t < 192) {
        apart = inputs[t] = channel_unit(columns1[t], e1);
    } else if (t < 320) {
        const int j = t - 192, both = hidden1[j] + (hidden2[j] = channel_unit(columns2[j], e2));
        atomicMax(&hidden[0], both);
        atomicMax(&hidden[1], -both);
    }
    const int inputs_apart = __syncthreads_or(apart);
    const int e = first ? e1 + hidden1[row] : e2 + hidden2[row];
    const int *columns = first ? inputs : outputs;
    unsigned head, tail;
    split_halves(times_power(v[0], kOperand - e - columns[k0]), times_power(v[1], kOperand - e - columns[k0 + 1]), head, tail);
    uint8_t *base = a.image + kCkHeader + (first ? (long long)chunk : 2ll * a.chunks) * kCkTile;
    const int place = half_place(row, k0 & 63);
    *reinterpret_cast<unsigned *>(base + place) = head;
    *reinterpret_cast<unsigned *>(base + (first ? a.chunks : 1) * kCkTile + place) = tail;
    if (blockIdx.x != 0) return;
    CkHeader *h = reinterpret_cast<CkHeader *>(a.image);
    if (t < 128) {
        h->hidden1[t] = (int8_t)hidden1[t];
        h->hidden2[t] = (int8_t)hidden2[t];
    }
    if (t < 192) h->inputs[t] = (int8_t)inputs[t];
    if (t < 64) h->outputs[t] = (int8_t)outputs[t];
    if (t == 0) {
        h->w1 = e1; h->w2 = e2; h->b1 = most[2] == 0 ? -1000 : binade(most[2]);
        h->hidden = hidden[0]; h->apart = (inputs_apart ? CK_INPUTS : 0) | (hidden[0] != -hidden[1] ? CK_HIDDEN : 0) | (outputs_apart ? CK_OUTPUTS : 0);
    }
}

// ---- what both kernels share ---------------------------------------------------------------------------------------------
// Operand of rows of 64 numbers with the summed index along the rows (MN-major): groups of eight rows 1024 bytes apart, the next 64
// columns `next_bytes` further.
__device__ inline uint64_t umma_desc_rows(unsigned smem_addr, unsigned next_bytes) {
    return (uint64_t)((smem_addr >> 4) & 0x3fffu) | ((uint64_t)((next_bytes >> 4) & 0x3fffu) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ inline void umma_f16(unsigned d_tmem, uint64_t a_desc, uint64_t b_desc, unsigned idesc, int accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// A from tensor memory: 128 lanes x 8 columns of two numbers.
__device__ inline void umma_f16_ts(unsigned d_tmem, unsigned a_tmem, uint64_t b_desc, unsigned idesc, int accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// M = 128, float16 x float16 -> 32 bits; `rows_b`: B is summed along its rows.
__device__ constexpr unsigned f16_idesc(int n, bool rows_b) {
    return (1u << 4) | (rows_b ? 1u << 16 : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
}

// What is worked out from `v` behind this is worked out again in every round of a loop: dozens of addresses kept over the tiles would
// take the registers of what is under way, and a spilled register comes back from L2 (shared memory leaves no L1).
__device__ __forceinline__ int worked_out_here(int v) {
    asm volatile("" : "+r"(v));
    return v;
}

struct CkArgs {
    const int8_t *codes;
    const uint8_t *exponents;
    const uint4 *mask;
    const float *dy, *b1;
    const uint8_t *image;
    float *dz, *partial;   // dz [rows, in]; partial [ctas][128][N1p + N2p], db1 in column `in`
    unsigned *dy_columns;  // [ctas][kCkProducers][64]: the largest finite magnitude of each column of dy in a warp's rows, the same in both kernels
    int looked;            // whether they are there (the weights' kernel looks for itself otherwise)
    const uint8_t *z_groups;  // [ctas][8]: the largest exponent of each group of z, in the same rows
    long long rows;
    int in, out, pitch, chunks, N1p, N2p, tiles;
    unsigned *status;
};

// Exponent field of the unit of a row from its largest finite magnitude (which is below 2 units; rows below 2^-112 have that unit), and
// 2^kOperand / unit.
__device__ __forceinline__ unsigned row_unit(unsigned largest) { return min(max(largest >> 23, kOperand + 1u), 254u); }
__device__ __forceinline__ float from_row_unit(unsigned field) { return __uint_as_float((254u + kOperand - field) << 23); }
// dh as it leaves its accumulator is below 48 (2^15)^2: times this it is an operand again.
constexpr int kDhDown = 21;
constexpr float kDhUnit = 1.f / (1 << kDhDown);

// One producer warp's 32 rows of dy, two neighbouring columns a lane: half a warp for a row of up to 32 columns, 24 lanes for one of up
// to 48 (TWO).  Loaded a tile ahead ...
template <bool TWO>
struct DyRows {
    static constexpr int kEach = TWO ? 1 : 2, kPasses = 32 / kEach;  // rows a pass
    float2 v[kPasses];
    __device__ __forceinline__ void load(const CkArgs &a, long long row0, int lane) {
        const int k = TWO ? 2 * lane : 2 * (lane & 15), r0 = TWO ? 0 : lane >> 4, out = worked_out_here(a.out);
        const float *p = a.dy + (row0 + r0) * a.out + k;
        const int rows = a.rows - row0 < 32 ? (int)(a.rows - row0) : 32;
        const bool one = k < a.out, two = k + 1 < a.out;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const bool there = r0 + i * kEach < rows;
            v[i].x = there && one ? __ldg(p + i * kEach * out) : 0.f;
            v[i].y = there && two ? __ldg(p + i * kEach * out + 1) : 0.f;
        }
    }
    __device__ __forceinline__ void put(uint8_t *heads, uint8_t *tails, int first, int i, float2 scale, int lane) const {
        unsigned head, tail;
        split_halves(v[i].x * scale.x, v[i].y * scale.y, head, tail);
        const int place = half_place(first + (TWO ? 0 : lane >> 4) + i * kEach, TWO ? 2 * lane : 2 * (lane & 15));  // (`first` is a multiple of 32)
        if (!TWO || lane < 24) {
            *reinterpret_cast<unsigned *>(heads + place) = head;
            *reinterpret_cast<unsigned *>(tails + place) = tail;
        }
    }
    // The columns in other units: units[] of 64, powers of two.
    __device__ __forceinline__ void times(const float *units, int lane) {
        const float2 f = reinterpret_cast<const float2 *>(units)[column(lane)];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            v[i].x *= f.x;
            v[i].y *= f.y;
        }
    }
    // ... and stored as heads and tails in units of their rows, whose exponents go to `units`: a lane works out one row's (four or two
    // lanes the same) and hands it round.
    __device__ __forceinline__ void store_by_row(uint8_t *heads, uint8_t *tails, int *units, int first, int lane, uint2 &most) const {
        constexpr int kLanes = TWO ? 32 : 16;
#pragma unroll
        for (int i0 = 0; i0 < kPasses; i0 += 8) {
            unsigned m[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned x = finite_magnitude(v[i0 + i].x), y = finite_magnitude(v[i0 + i].y);
                most = make_uint2(max(most.x, x), max(most.y, y));
                m[i] = max(x, y);
            }
            const unsigned field = row_unit(gather_max8<kLanes>(m));
            const float scale = from_row_unit(field);
            const int pass = i0 + (lane & (kLanes - 1)) / (kLanes / 8);
            if (lane % (kLanes / 8) == 0) units[first + (TWO ? 0 : lane >> 4) + pass * kEach] = (int)field - 127;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = __shfl_sync(kFull, scale, max8_lane<kLanes>(i));
                put(heads, tails, first, i0 + i, make_float2(u, u), lane);
            }
        }
    }
    // The largest of a lane's two columns (in `units`, where they are in any) to memory as they were, [32] pairs a warp.
    static __device__ __forceinline__ void put_columns(unsigned *to, uint2 most, const float *units, int lane) {
        if (!TWO) most = make_uint2(max(most.x, __shfl_xor_sync(kFull, most.x, 16)), max(most.y, __shfl_xor_sync(kFull, most.y, 16)));
        if (units) {
            const float2 f = reinterpret_cast<const float2 *>(units)[column(lane)];
            most = make_uint2(finite_magnitude(__uint_as_float(most.x) / f.x), finite_magnitude(__uint_as_float(most.y) / f.y));
        }
        reinterpret_cast<uint2 *>(to)[lane] = TWO || lane < 16 ? most : make_uint2(0, 0);
    }
    // The largest finite magnitude of the warp's rows with the columns times `f`; and heads and tails of the columns times `scale`.
    __device__ __forceinline__ unsigned largest(float2 f) const {
        unsigned x = 0, y = 0;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            x = max(x, finite_magnitude(v[i].x));
            y = max(y, finite_magnitude(v[i].y));
        }
        return warp_max(max(finite_magnitude(__uint_as_float(x) * f.x), finite_magnitude(__uint_as_float(y) * f.y)));
    }
    __device__ __forceinline__ void store(uint8_t *heads, uint8_t *tails, float2 scale, int first, int lane) const {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) put(heads, tails, first, i, scale, lane);
    }
    static __device__ __forceinline__ int column(int lane) { return TWO ? lane : lane & 15; }  // this lane's pair of columns
};

__device__ __forceinline__ void ck_copy_image(uint8_t *dst, const uint8_t *image, int chunks, uint64_t *bar) {
    const int tiles = 2 * chunks + 2;
    mbar_arrive_expect(bar, (unsigned)(tiles * kCkTile));
    for (int q = 0; q < tiles; ++q) bulk_copy_g2s(dst + q * kCkTile, image + kCkHeader + (long long)q * kCkTile, kCkTile, bar);
}

// Channels of the image in other units, once in front of the tiles (a copy has landed, the MMAs have not begun): the rows are multiplied by
// row[] and the columns by column[], powers of two (NULL: 1).  Only where channels lie apart: a microsecond or two for the 128 KB of 163 inputs.
__device__ __noinline__ void ck_rescale(uint8_t *heads, uint8_t *tails, int chunks, const float *row, const float *column, int threads) {
    for (int q = threadIdx.x % threads; q < chunks * 128 * 8; q += threads) {
        const int r = (q >> 3) & 127, k = (q >> 10) * 64 + (((q & 7) ^ (r & 7)) << 3);
        const float f = row ? row[r] : 1.f;
        uint4 head = reinterpret_cast<uint4 *>(heads)[q], tail = reinterpret_cast<uint4 *>(tails)[q];
        unsigned h[4] = {head.x, head.y, head.z, head.w}, l[4] = {tail.x, tail.y, tail.z, tail.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpack_halves(h[i]), b = unpack_halves(l[i]);  // (the sum is exact: 22 bits)
            split_halves((a.x + b.x) * (column ? f * column[k + 2 * i] : f), (a.y + b.y) * (column ? f * column[k + 2 * i + 1] : f), h[i], l[i]);
        }
        reinterpret_cast<uint4 *>(heads)[q] = make_uint4(h[0], h[1], h[2], h[3]);
        reinterpret_cast<uint4 *>(tails)[q] = make_uint4(l[0], l[1], l[2], l[3]);
    }
}
// The eight warps of the epilogue of dz's and the weights' kernel, which see to the units; never inside a loop that a bounded wait may leave.
constexpr int kCkEpilogue = 256;
__device__ __forceinline__ void ck_epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kCkEpilogue) : "memory"); }
__device__ __forceinline__ float channel_factor(int e) { return power_of_two(max(e, -126)); }

// ---- dz ----------------------------------------------------------------------------------------------------------------
// Warp-specialised, one persistent CTA per SM, tiles of 128 rows: four producer warps (32 rows of dy each, a tile ahead in registers;
// a lane of the first issues the MMAs), eight that mask dh and take it apart in place (lane = row; head and tail of 16 columns fill the
// 16 columns of the accumulator they came from) and store dz of the tile before.  dh has two accumulators, so that the next tile's is made
// meanwhile.
struct CkDzShared {
    uint64_t image, units_known, op_full, op_empty, dh_full[2], dh_ready[2], dz_full, dz_empty, staged[4], copied[4];
    int units[kCkRowRing][kCkRows];
    alignas(8) float outputs[64], inputs[192];  // units of W2's and W1's columns
    float hidden[128];                          // what a hidden unit weighs against the largest
    uint32_t tmem_base;
    int abort;
};
constexpr int kCkDzCol = 256;
// A quarter's 32 rows of dz are put together as they lie in memory; two quarters share a buffer where four do not fit.  (dz alone of
// 262,144 rows, four / two buffers: 100 columns 56.2 / 63.3 us; 66, 67 and 128 the same.)
__host__ __device__ constexpr int ck_dz_buffers(int in) { return in <= 128 ? 4 : 2; }
static int ck_dz_smem(int chunks, int in) { return 1024 + (2 * chunks + 2) * kCkTile + 2 * kCkTile + ck_dz_buffers(in) * 128 * in; }
__device__ inline void bulk_copy_s2g(void *dst, const void *src, unsigned bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}
__device__ inline void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ inline void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ inline void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// PIECES: rows of a multiple of four columns leave by 16 bytes (put_16_pieces): 262,144 rows of 128 and 160 columns 191 -> 76 and 215 -> 84 us.  An
// argument of the kernel: with both ways in one the registers of the other widths suffered (82 -> 89 us for 163).
template <bool TWO, bool PIECES>
__global__ void __launch_bounds__(kCkThreads, 1) mlp_checkpoint_dz_kernel(const __grid_constant__ CkArgs a) {
    after_previous_kernel();
    extern __shared__ uint8_t ck_raw[];
    __shared__ CkDzShared sh;
    uint8_t *base = ck_raw + ((1024u - (smem_u32(ck_raw) & 1023u)) & 1023u);
    uint8_t *w2 = base + 2 * a.chunks * kCkTile, *ops = w2 + 2 * kCkTile;  // ops: heads | tails
    float *staged = reinterpret_cast<float *>(ops + 2 * kCkTile);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&sh.image, 1);
        mbar_init(&sh.op_full, kCkProducers);
        mbar_init(&sh.op_empty, 1);
        for (int q = 0; q < 2; ++q) {
            mbar_init(&sh.dh_full[q], 1);
            mbar_init(&sh.dh_ready[q], 8);
        }
        for (int q = 0; q < 4; ++q) {
            mbar_init(&sh.staged[q], 2);
            mbar_init(&sh.copied[q], 1);
        }
        mbar_init(&sh.dz_full, 2);  // the products, and the MMA lane itself: what it has seen of the producers' writes the epilogue sees
        mbar_init(&sh.dz_empty, 8);
        mbar_init(&sh.units_known, 8);
        sh.abort = 0;
        mbar_fence_init();
    }
    const CkHeader &units = *reinterpret_cast<const CkHeader *>(a.image);
    const int apart = units.apart;  // (looked at behind the barrier)
    if (warp == kCkProducer0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = sh.tmem_base;
    const int ntile = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    auto row_of = [&](int it) { return ((long long)blockIdx.x + (long long)it * gridDim.x) * kCkRows; };
    bool ok = true;

    if (warp >= kCkProducer0) {
        // the first of the producers issues the MMAs as well (one lane): dh of a tile as soon as its operands are there, then dz of the
        // tile before
        const bool issues = warp == kCkProducer0;
        const int mine = (warp - kCkProducer0) * 32;
        if (issues && lane == 0) ck_copy_image(base, a.image, a.chunks, &sh.image);
        const unsigned id1 = f16_idesc(128, false), id2 = f16_idesc((a.in + 15) / 16 * 16, true);
        const int ks1 = (a.out + 15) / 16;
        const uint64_t w2h = umma_desc(smem_u32(w2)), w2l = umma_desc(smem_u32(w2 + kCkTile));
        const unsigned w1h = smem_u32(base), w1l = smem_u32(base + a.chunks * kCkTile);
        auto first = [&](int t) -> bool {
            const int b = t & 1;
            if (t == 0 && !umma_wait(&sh.image, 0, &sh.abort)) return false;
            if (!umma_wait(&sh.op_full, t & 1, &sh.abort)) return false;
            if (t > 1 && !umma_wait(&sh.dz_full, t & 1, &sh.abort)) return false;  // this accumulator was the operand of tile t - 2
            tc_fence_after();
            const uint64_t dh = umma_desc(smem_u32(ops)), dl = umma_desc(smem_u32(ops + kCkTile));
            const unsigned d = tmem + b * 128;
            for (int ks = 0; ks < ks1; ++ks) {  // the small products first: an addition cuts off what lies below the sum's last bit
                umma_f16(d, dl + 2 * ks, w2h + 2 * ks, id1, ks != 0);
                umma_f16(d, dh + 2 * ks, w2l + 2 * ks, id1, 1);
            }
            for (int ks = 0; ks < ks1; ++ks) umma_f16(d, dh + 2 * ks, w2h + 2 * ks, id1, 1);
            umma_commit(&sh.op_empty);
            umma_commit(&sh.dh_full[b]);
            return true;
        };
        auto second = [&](int t) -> bool {
            const int b = t & 1;
            if (!umma_wait(&sh.dh_ready[b], (t >> 1) & 1, &sh.abort)) return false;
            if (!umma_wait(&sh.dz_empty, (t & 1) ^ 1, &sh.abort)) return false;
            tc_fence_after();
            const unsigned d = tmem + kCkDzCol, ah = tmem + b * 128;
            for (int ks = 0; ks < 8; ++ks) {  // 16 hidden units: 2048 bytes of W1's rows
                umma_f16_ts(d, ah + 16 * ks + 8, umma_desc_rows(w1h + 2048 * ks, kCkTile), id2, ks != 0);
                umma_f16_ts(d, ah + 16 * ks, umma_desc_rows(w1l + 2048 * ks, kCkTile), id2, 1);
            }
            for (int ks = 0; ks < 8; ++ks) umma_f16_ts(d, ah + 16 * ks, umma_desc_rows(w1h + 2048 * ks, kCkTile), id2, 1);
            umma_commit(&sh.dz_full);
            mbar_arrive(&sh.dz_full);
            return true;
        };
        DyRows<TWO> rows;
        uint2 most = make_uint2(0, 0);
        if (ntile > 0) rows.load(a, row_of(0) + mine, lane);
        if (apart) ok = umma_wait(&sh.units_known, 0, &sh.abort);
#pragma unroll 1
        for (int t = 0; t < ntile && ok; ++t) {
            if (!(ok = umma_wait(&sh.op_empty, (t & 1) ^ 1, &sh.abort))) break;
            if (apart & CK_OUTPUTS) rows.times(sh.outputs, lane);
            rows.store_by_row(ops, ops + kCkTile, sh.units[t % kCkRowRing], mine, lane, most);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.op_full);
                if (issues) ok = first(t);
            }
            __syncwarp();
            if (t + 1 < ntile) rows.load(a, row_of(t + 1) + mine, lane);
            if (issues) {
                if (lane == 0) {
                    ok = ok && (t == 0 || second(t - 1));
                    if (ok && t + 1 == ntile) ok = second(t);
                }
                ok = __shfl_sync(kFull, (int)ok, 0) != 0;
            }
        }
        rows.put_columns(a.dy_columns + (blockIdx.x * kCkProducers + warp - kCkProducer0) * 64, most, apart & CK_OUTPUTS ? sh.outputs : nullptr, lane);
        if (!ok && lane == 0) {
            atomicOr(a.status, issues ? CK_STATUS_MMA : CK_STATUS_PRODUCER);
            __nanosleep(20000);  // copies in flight land before the CTA leaves
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2;  // rows 32 quarter + lane; hidden units 64 half and up, every second 16 columns of dz
        const unsigned tlane = tmem + ((unsigned)(quarter * 32) << 16);
        if (apart) {
            if (threadIdx.x < 64) sh.outputs[threadIdx.x] = channel_factor(units.outputs[threadIdx.x]);
            if (threadIdx.x < 192) sh.inputs[threadIdx.x] = channel_factor(units.inputs[threadIdx.x]);
            if (threadIdx.x < 128) sh.hidden[threadIdx.x] = channel_factor(units.hidden1[threadIdx.x] + units.hidden2[threadIdx.x] - units.hidden);
            ck_epilogue_barrier();
            if (apart & CK_HIDDEN) {  // dh with what its hidden unit weighs in dz
                umma_wait(&sh.image, 0, &sh.abort);
                ck_rescale(w2, w2 + kCkTile, 1, sh.hidden, nullptr, kCkEpilogue);
                fence_proxy_async();
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(&sh.units_known);
        }
        const int unit_of_w = units.w1 + units.w2 + units.hidden + kDhDown - 3 * kOperand;
        const int buffers = ck_dz_buffers(a.in);  // (with two of them quarters 0 and 2, 1 and 3 take turns)
        float *stg = staged + quarter % buffers * 32 * a.in;
        const bool aligned = (uintptr_t)a.dz % 16 == 0;
        auto bits_of = [&](int t) {
            const long long row = row_of(t) + quarter * 32 + lane;
            return row < a.rows ? __ldg(reinterpret_cast<const uint2 *>(a.mask) + 2 * row + half) : make_uint2(0, 0);
        };
        auto leave = [&](int t) -> bool {  // dz of tile t
            const long long row0 = row_of(t) + quarter * 32;
            const int nrows = a.rows - row0 < 32 ? (int)(a.rows - row0) : 32;  // may be <= 0
            if (!umma_wait(&sh.dz_full, t & 1, &sh.abort)) return false;
            tc_fence_after();
            // the row's unit times those of the weights: one power of two unless it is out of range
            const int e = sh.units[t % kCkRowRing][quarter * 32 + lane] + unit_of_w, e1 = max(min(e, 127), -126);
            const float unit = power_of_two(e1), rest = power_of_two(max(e - e1, -126));
            const bool far = __any_sync(kFull, e != e1) || (apart & CK_INPUTS);
            float *row = stg + lane * a.in;
            auto emptied = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.dz_empty);
            };
            // The rows that were here before have left: this quarter's, and those of the one that shares its buffer.  (A barrier each, one
            // phase a tile: a wait tells a barrier's last two phases apart and no more.)
            auto free_again = [&]() -> bool {
                if (t > 0 && !umma_wait(&sh.copied[quarter], (t - 1) & 1, &sh.abort)) return false;
                if (buffers == 4) return true;
                if (quarter >= 2) return umma_wait(&sh.copied[quarter - 2], t & 1, &sh.abort);
                return t == 0 || umma_wait(&sh.copied[quarter + 2], (t - 1) & 1, &sh.abort);
            };
            auto put = [&](unsigned(&r)[16], int c0, auto full) {
                if constexpr (PIECES) {
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]) * unit;
                    put_16_pieces(row + c0, decltype(full)::value ? 16 : a.in - c0, first_piece(a.in, lane), v);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (decltype(full)::value || c0 + j < a.in) row[c0 + j] = __uint_as_float(r[j]) * unit;
                }
            };
            if (!free_again()) return false;
            auto block = [&](int c0, auto full) {
                unsigned r[16];
                tmem_ld16(tlane + kCkDzCol + c0, r);
                tc_wait_ld();
                put(r, c0, full);
            };
            int c0 = 16 * half;
#pragma unroll 1
            for (; c0 + 16 <= a.in; c0 += 32) block(c0, std::true_type());
            if (c0 < a.in) block(c0, std::false_type());
            emptied();
            if (far)  // (this thread's own)
#pragma unroll 1
                for (c0 = 16 * half; c0 < a.in; c0 += c0 % 16 == 15 ? 17 : 1) row[c0] *= rest * (apart & CK_INPUTS ? sh.inputs[c0] : 1.f);
            fence_proxy_async();  // the copy reads these
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.staged[quarter]);
            if (half == 0) {
                if (!umma_wait(&sh.staged[quarter], t & 1, &sh.abort)) return false;
                if (nrows == 32 && aligned) {
                    if (lane == 0) {
                        bulk_copy_s2g(a.dz + row0 * a.in, stg, (unsigned)(128 * a.in));
                        bulk_commit();
                        bulk_wait_read();
                    }
                } else {
                    for (int q = lane; q < nrows * a.in; q += 32) a.dz[row0 * a.in + q] = stg[q];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.copied[quarter]);
            }
            return true;
        };
        uint2 next = ntile > 0 ? bits_of(0) : make_uint2(0, 0);
#pragma unroll 1
        for (int t = 0; t < ntile; ++t) {
            const int b = t & 1;
            const uint2 m = next;
            if (t + 1 < ntile) next = bits_of(t + 1);
            if (!(ok = umma_wait(&sh.dh_full[b], (t >> 1) & 1, &sh.abort))) break;
            tc_fence_after();
            const unsigned d = tlane + b * 128 + 64 * half;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const unsigned word = c < 2 ? m.x : m.y, bits = c & 1 ? word >> 16 : word;
                unsigned r[16], parts[16];
                tmem_ld16(d + 16 * c, r);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    split_halves(bits >> (2 * j) & 1u ? __uint_as_float(r[2 * j]) * kDhUnit : 0.f,
                                 bits >> (2 * j + 1) & 1u ? __uint_as_float(r[2 * j + 1]) * kDhUnit : 0.f, parts[j], parts[8 + j]);
                tmem_st16(d + 16 * c, parts);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.dh_ready[b]);
            if (t > 0 && !(ok = leave(t - 1))) break;
        }
        if (ok && ntile > 0) ok = leave(ntile - 1);
        if (lane == 0) bulk_wait();  // the rows are in memory before the block ends
        if (!ok && lane == 0) atomicOr(a.status, CK_STATUS_EPILOGUE);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kCkProducer0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- the weights' gradients -----------------------------------------------------------------------------------------------
// The same tiles with lane = hidden unit: zh W1^T and dy W2 come out transposed, masked and taken apart in place they are the A operands
// of the sums over the tile's rows.  The bits of 32 units and a row are one word, the same for a warp.  A tile's sums leave the
// accumulators with the tile's unit and are added in 32 bits, in registers: up to 7 blocks of 16 columns a thread (kBlocks).
//
// A tile's way at 163 inputs and 35 outputs, in clocks of 16,000: dy into heads and tails 2,200, dh 1,300, zh W1^T 3,300 with dh's mask
// meanwhile, its own mask 1,900 with dW1's products meanwhile, dW2's products 1,700 with the next zh (2,400) meanwhile.  In the order zh,
// dy, products, masks, sums it was 24,000.
struct CkWeightsShared {
    uint64_t image, units, op_full, z_empty, dy_empty, dy_known, dh_full, pre_full, dh_ready, pre_ready, g1_full, g2_full;
    alignas(16) unsigned mask[4][kCkRows];
    unsigned dy_most[2][kCkProducers];     // of two tiles: largest finite magnitude of each producer's rows
    int dy_unit;
    alignas(16) uint8_t exponents[kCkRows * 6];
    float both[kCkRows];
    int z_unit;
    // of this CTA's rows: the largest finite dy of each column, the largest exponent of each group of z, the magnitudes of each column's codes
    // (a byte each, whose first bit is that of the largest); and what follows from them (ck_settle)
    unsigned dy_columns[64], z_groups[8], used[44];
    alignas(8) float inputs[192], outputs[64];  // factors of the image's columns
    alignas(8) float dy_units[64], dy_back[64];
    float z_back[8];
    unsigned z_shift[kCkRows * 6 / 4];  // what a tile's exponents are moved by, four a word
    uint8_t z_move[8];
    float2 back[2][128];
    int add1, add2, most1;  // exponents of the units of W1 and W2 (of dh as it leaves its accumulator), and of the largest of zh W1^T's products
    int apart, least_field, settle;
    uint32_t tmem_base;
    int abort;
};
constexpr int kCkPreCol = 0, kCkDhCol = 128, kCkW1Col = 256, kCkW2Col = 448;
static int ck_weights_smem(int chunks) { return 1024 + (2 * chunks + 2) * kCkTile + chunks * kCkTile + 2 * kCkTile; }

// Sixteen codes as numbers of float16 in units of 2^-8 of the tile's: exact while they are normal or fit the subnormal ones.
__device__ __forceinline__ void decode_codes(const uint4 &q, __half2 scale, uint4 &lo, uint4 &hi) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    unsigned out[8];
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1024 + 128
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned u = w[i] ^ 0x80808080u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const unsigned p = __byte_perm(u, 0x64646464u, j ? 0x4342 : 0x4140);  // 0x64uu: 1024 + code + 128
            const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2 *>(&p), bias), scale);
            out[2 * i + j] = *reinterpret_cast<const unsigned *>(&v);
        }
    }
    lo = make_uint4(out[0], out[1], out[2], out[3]);
    hi = make_uint4(out[4], out[5], out[6], out[7]);
}

// A gradient of W2 sums one column of dy, and one of W1 a group of z's: neither has to do with the size of the others.  So a column of dy, and a
// group of z, whose largest in this CTA's rows lies far below the largest of all has a unit of its own: it is multiplied by a power of two,
// the image's column by the inverse (dh and zh W1^T sum over them), and the power comes back when the CTA's sums leave.  Columns of W1 come out
// of their own units on the same way, in the unit of the largest that meets a code (a column whose codes are all zero has no size).
// The epilogue's warps see to this in front of the tiles, while the producers have the first one's loads on their way.  The sizes are those
// that the forward (groups of z) and dz's kernel (columns of dy) saw in the same rows; where dz was not asked for dy is read once more (148 ->
// 164 us for 262,144 rows of 163 and 35), and so are the codes where columns of W1 lie apart.  Where nothing does it is a few instructions
// (ck_apart): all that runs once a CTA comes from memory, and the whole of it, always run, cost 3 us.
constexpr int kGroupsApart = 16, kGroupsFarthest = 120;  // zh is exact 2^32 below the largest of its tile: 2^16 are left to the rows
enum { CK_APART_W1 = 1, CK_APART_W2 = 2, CK_APART_Z = 4 };
// Whether anything lies apart; a warp's lanes hold the columns `lane` and `lane` + 32 of dy, and eight of them the groups of z.
__device__ __forceinline__ bool ck_apart(const CkArgs &a, int header, unsigned column, unsigned further, unsigned group) {
    auto field = [](unsigned m) { return (int)max(m >> 23, 1u); };
    const unsigned all = __reduce_max_sync(kFull, max(column, further)), least = __reduce_min_sync(kFull, min(column ? column : ~0u, further ? further : ~0u));
    const unsigned most = __reduce_max_sync(kFull, group), small = __reduce_min_sync(kFull, group ? group : ~0u);
    return (header & (CK_INPUTS | CK_OUTPUTS)) || !a.looked || (all && field(all) - field(least) >= kApart) || (most && most - small >= kGroupsApart);
}
// The units of a CTA where something does, by the epilogue's threads; ends with their barrier.
__device__ __forceinline__ void ck_settle(CkWeightsShared &sh, const CkArgs &a, uint8_t *base, int ntile) {
    const CkHeader &head = *reinterpret_cast<const CkHeader *>(a.image);
    const int t = threadIdx.x, lane = t & 31, out = a.out, units = a.pitch / 16, header = head.apart;
    const long long row0 = (long long)blockIdx.x * kCkRows, rows_on = (long long)gridDim.x * kCkRows;  // of this CTA's first tile, to the next
    if (t < 64) sh.dy_columns[t] = 0;
    if (t < 44) sh.used[t] = 0;
    if (t < 8) sh.z_groups[t] = __ldg(a.z_groups + blockIdx.x * 8 + t);
    if (t == 0) sh.add1 = sh.add2 = sh.most1 = -1000;  // (what comes to the matrices' exponents, which are added last)
    ck_epilogue_barrier();
    if (a.looked) {
        atomicMax(&sh.dy_columns[t % 64], __ldg(a.dy_columns + blockIdx.x * kCkProducers * 64 + t));
    } else {  // a thread goes on by a multiple of the columns, so that it stays in the same ones
        const int turn = kCkEpilogue / out * out, each = 32 * out, total = ntile * each;
        const long long end = a.rows * out;
        unsigned m[4] = {};
        if (t < turn) {
#pragma unroll 8
            for (int i = t; i < total; i += turn) {
                const int tile = i / each;
                const long long at = (row0 + tile * rows_on) * out + 4 * (i - tile * each);
                const float4 v = at + 4 <= end ? __ldg(reinterpret_cast<const float4 *>(a.dy + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
                m[0] = max(m[0], finite_magnitude(v.x));
                m[1] = max(m[1], finite_magnitude(v.y));
                m[2] = max(m[2], finite_magnitude(v.z));
                m[3] = max(m[3], finite_magnitude(v.w));
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) atomicMax(&sh.dy_columns[(4 * t + q) % out], m[q]);
        }
        const bool last = ntile > 0 && row0 + (ntile - 1) * rows_on + kCkRows >= a.rows;  // this CTA's rows end with the last one
        if (last && t < (int)(end & 3)) atomicMax(&sh.dy_columns[((end & ~3ll) + t) % out], finite_magnitude(__ldg(a.dy + (end & ~3ll) + t)));
    }
    if (header & CK_INPUTS) {
        const int turn = kCkEpilogue / units * units, each = kCkRows * units, total = ntile * each;
        uint4 any = make_uint4(0, 0, 0, 0);
        if (t < turn) {
#pragma unroll 4
            for (int i = t; i < total; i += turn) {
                const int tile = i / each;
                const long long at = (row0 + tile * rows_on) * units + (i - tile * each);
                const uint4 v = at < a.rows * units ? __ldg(reinterpret_cast<const uint4 *>(a.codes) + at) : make_uint4(0, 0, 0, 0);
                any.x |= __vabs4(v.x); any.y |= __vabs4(v.y); any.z |= __vabs4(v.z); any.w |= __vabs4(v.w);
            }
            const int u = t % units;
            atomicOr(&sh.used[4 * u], any.x);
            atomicOr(&sh.used[4 * u + 1], any.y);
            atomicOr(&sh.used[4 * u + 2], any.z);
            atomicOr(&sh.used[4 * u + 3], any.w);
        }
    }
    ck_epilogue_barrier();
    int mine = 0;
    bool counts = false;
    if (t < 64) {
        const unsigned all = warp_max(max(sh.dy_columns[lane], sh.dy_columns[lane + 32]));  // (columns that do not exist are zero)
        const int p = channel_unit(sh.dy_columns[t], binade(all));
        sh.dy_units[t] = power_of_two(-p);
        sh.dy_back[t] = power_of_two(p);
        counts = t < out;
        mine = p + head.outputs[t];
        if (counts) atomicMax(&sh.add2, mine);
        if (p) atomicMax(&sh.least_field, kOperand + 1 - p);  // (no power of two leaves 32 bits)
    } else {
        const int k = t - 64, g = k / 32;
        const unsigned all = warp_max(sh.z_groups[lane & 7]);
        const int far = (int)sh.z_groups[g] - (int)all, q = sh.z_groups[g] == 0 || far > -kGroupsApart ? 0 : max(far, -kGroupsFarthest);
        if (k % 32 == 0) {
            sh.z_back[g] = channel_factor(q);
            sh.z_move[g] = (uint8_t)-q;
            if (q) atomicOr(&sh.apart, CK_APART_Z);
        }
        const unsigned codes = !(header & CK_INPUTS) ? 127u : k < a.in ? sh.used[k / 4] >> (8 * (k % 4)) & 0xffu : 0u;
        counts = k < a.in && codes != 0;
        mine = q + head.inputs[k];
        if (counts) {
            atomicMax(&sh.add1, mine);
            atomicMax(&sh.most1, mine - (__clz(codes) - 25));
        }
    }
    ck_epilogue_barrier();
    if (t == 64 && sh.add1 == -1000) sh.add1 = sh.most1 = 0;  // (no column has a code)
    if (t < 64) {
        sh.outputs[t] = counts ? channel_factor(mine - sh.add2) : 0.f;
        if (counts && mine != sh.add2) atomicOr(&sh.apart, CK_APART_W2);
    } else {
        sh.inputs[t - 64] = counts ? channel_factor(mine - sh.add1) : 0.f;
        if (counts && mine != sh.add1) atomicOr(&sh.apart, CK_APART_W1);
    }
    if (sh.apart & CK_APART_Z)
        for (int b = t; b < kCkRows * 6; b += kCkEpilogue) reinterpret_cast<uint8_t *>(sh.z_shift)[b] = sh.z_move[b % ((a.in + 31) / 32)];
    ck_epilogue_barrier();
    uint8_t *w2 = base + 2 * a.chunks * kCkTile;
    if (sh.apart & (CK_APART_W1 | CK_APART_W2)) {
        umma_wait(&sh.image, 0, &sh.abort);
        if (sh.apart & CK_APART_W1) ck_rescale(base, base + a.chunks * kCkTile, a.chunks, nullptr, sh.inputs, kCkEpilogue);
        if (sh.apart & CK_APART_W2) ck_rescale(w2, w2 + kCkTile, 1, nullptr, sh.outputs, kCkEpilogue);
        fence_proxy_async();
    }
    if (t == 0) {
        sh.add1 += head.w1;
        sh.most1 += head.w1;
        sh.add2 += head.w2 + kDhDown - 2 * kOperand;
    }
    ck_epilogue_barrier();
}

template <int kBlocks, bool TWO>
__global__ void __launch_bounds__(kCkThreads, 1) mlp_checkpoint_weights_kernel(const __grid_constant__ CkArgs a) {
    after_previous_kernel();
    extern __shared__ uint8_t ck_raw[];
    __shared__ CkWeightsShared sh;
    uint8_t *base = ck_raw + ((1024u - (smem_u32(ck_raw) & 1023u)) & 1023u);
    uint8_t *w2 = base + 2 * a.chunks * kCkTile, *zt = w2 + 2 * kCkTile, *dyt = zt + a.chunks * kCkTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&sh.image, 1);
        mbar_init(&sh.op_full, kCkProducers);
        mbar_init(&sh.z_empty, 1);
        mbar_init(&sh.dy_empty, 1);
        mbar_init(&sh.dy_known, kCkProducers);
        mbar_init(&sh.dh_full, 2);  // the products, and the MMA lane itself: what it has seen of the producers' writes the epilogue sees
        mbar_init(&sh.pre_full, 1);
        mbar_init(&sh.dh_ready, 8);
        mbar_init(&sh.pre_ready, 8);
        mbar_init(&sh.g1_full, 1);
        mbar_init(&sh.g2_full, 1);
        mbar_init(&sh.units, 8);
        sh.abort = 0;
        mbar_fence_init();
    }
    const CkHeader &head = *reinterpret_cast<const CkHeader *>(a.image);
    unsigned column = 0, further = 0, group = 0;  // (what is loaded here is looked at behind the barrier)
    int header = 0, w1 = 0, w2_unit = 0;
    if (warp == 0) {
        header = head.apart; w1 = head.w1; w2_unit = head.w2 + kDhDown - 2 * kOperand;
        if (a.looked) {
            const unsigned *p = a.dy_columns + blockIdx.x * kCkProducers * 64 + lane;
            column = max(max(__ldg(p), __ldg(p + 64)), max(__ldg(p + 128), __ldg(p + 192)));
            further = max(max(__ldg(p + 32), __ldg(p + 96)), max(__ldg(p + 160), __ldg(p + 224)));
        }
        if (lane < 8) group = __ldg(a.z_groups + blockIdx.x * 8 + lane);
    }
    static_assert(kCkProducers == 4, "as read here");
    if (threadIdx.x < 64) sh.dy_units[threadIdx.x] = sh.dy_back[threadIdx.x] = 1.f;
    else if (threadIdx.x < 72) sh.z_back[threadIdx.x - 64] = 1.f;
    else if (threadIdx.x == 72) sh.apart = 0, sh.least_field = kOperand + 1;
    if (warp == kCkProducer0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = sh.tmem_base;
    const int ntile = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    auto row_of = [&](int it) { return ((long long)blockIdx.x + (long long)it * gridDim.x) * kCkRows; };
    bool ok = true;

    if (warp >= kCkProducer0) {
        // the first of the producers issues the products that make the A operands (one lane)
        const bool issues = warp == kCkProducer0;
        if (issues && lane == 0) ck_copy_image(base, a.image, a.chunks, &sh.image);
        // (operands are described where they are used: kept over the loop they would cost the producers their registers, and a spilled
        // register comes back from L2)
        const int chunks = a.chunks;
        // MMAs into one accumulator follow one another: changing it after each costs half as much again (zh W1^T and dh in turn 5,000 clocks
        // instead of 3,400 at 163 inputs and 35 outputs).
        auto before = [&](int t) -> bool {  // dh and zh W1^T of tile t
            if (t == 0 && !umma_wait(&sh.image, 0, &sh.abort)) return false;
            if (!umma_wait(&sh.op_full, t & 1, &sh.abort)) return false;
            tc_fence_after();
            // (the A operands of tile t - 1 lay where these go: the producers have waited for both of its sums)
            const int ks1 = (a.in + 15) / 16, ks2 = (a.out + 15) / 16;
            const unsigned id = f16_idesc(128, false);
            const uint64_t w1h = umma_desc(smem_u32(base)), w1l = umma_desc(smem_u32(base + chunks * kCkTile));
            const uint64_t w2h = umma_desc(smem_u32(w2)), w2l = umma_desc(smem_u32(w2 + kCkTile));
            const uint64_t zk = umma_desc(smem_u32(zt)), dyh = umma_desc(smem_u32(dyt)), dyl = umma_desc(smem_u32(dyt + kCkTile));
            auto k = [](int ks) { return (uint64_t)((ks >> 2) * (kCkTile >> 4) + 2 * (ks & 3)); };  // 16 columns further
            const unsigned pre = tmem + kCkPreCol, dh = tmem + kCkDhCol;
            for (int ks = 0; ks < ks2; ++ks) {
                umma_f16(dh, w2l + 2 * ks, dyh + 2 * ks, id, ks != 0);
                umma_f16(dh, w2h + 2 * ks, dyl + 2 * ks, id, 1);
            }
            for (int ks = 0; ks < ks2; ++ks) umma_f16(dh, w2h + 2 * ks, dyh + 2 * ks, id, 1);
            umma_commit(&sh.dh_full);
            mbar_arrive(&sh.dh_full);
            for (int ks = 0; ks < ks1; ++ks) umma_f16(pre, w1l + k(ks), zk + k(ks), id, ks != 0);
            for (int ks = 0; ks < ks1; ++ks) umma_f16(pre, w1h + k(ks), zk + k(ks), id, 1);
            umma_commit(&sh.pre_full);
            return true;
        };
        const int first = (warp - kCkProducer0) * 32, groups = (a.in + 31) / 32, units = a.pitch / 16;  // units of 16 codes in a row
        const unsigned per_unit = 65535u / units + 1;  // q / units = q * per_unit >> 16 for q < 352
        DyRows<TWO> rows;
        uint4 mask;
        constexpr int kUnits = 11;
        uint4 code[kUnits];
        constexpr int kWords = 6;
        unsigned exps[kWords];  // the whole tile's, four a word: each warp finds the largest for itself
        auto load = [&](int t) {
            const long long row0 = row_of(t) + first;
            {
                const long long tile0 = row_of(t);
                const int bytes = (int)(a.rows - tile0 < kCkRows ? a.rows - tile0 : kCkRows) * groups;
                const uint8_t *p = a.exponents + tile0 * groups;
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const int q = 4 * (i * 32 + lane);
                    unsigned w = 0;
                    if (q + 4 <= bytes) {
                        w = __ldg(reinterpret_cast<const unsigned *>(p + q));
                    } else {
#pragma unroll
                        for (int j = 0; j < 3; ++j)
                            if (q + j < bytes) w |= (unsigned)__ldg(p + q + j) << (8 * j);
                    }
                    exps[i] = w;
                }
            }
            rows.load(a, row0, lane);
            mask = row0 + lane < a.rows ? __ldg(a.mask + row0 + lane) : make_uint4(0, 0, 0, 0);
            const int lane0 = worked_out_here(lane);
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {  // flat, so that lines are read whole
                const int q = i * 32 + lane0;
                code[i] = q < 32 * units && row0 + (q * per_unit >> 16) < a.rows ? __ldg(reinterpret_cast<const uint4 *>(a.codes + row0 * a.pitch) + q) : make_uint4(0, 0, 0, 0);
            }
        };
        if (ntile > 0) load(0);
        ok = umma_wait(&sh.units, 0, &sh.abort);
        const int apart = sh.apart;
#pragma unroll 1
        for (int t = 0; t < ntile && ok; ++t) {
            if (apart & CK_APART_Z) {  // exponents in units of their groups (neither 255 nor a byte that does not exist)
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const unsigned keep = __vcmpeq4(exps[i], 0xffffffffu) | __vcmpeq4(exps[i], 0u);
                    exps[i] = __vaddus4(exps[i], sh.z_shift[i * 32 + lane] & ~keep);
                }
            }
            unsigned most = 0x07070707u;
#pragma unroll
            for (int i = 0; i < kWords; ++i) most = __vmaxu4(most, exps[i] & ~__vcmpeq4(exps[i], 0xffffffffu));
            most = __vmaxu4(most, most >> 16);
            const int largest = (int)warp_max(max(most & 0xffu, most >> 8 & 0xffu));
            // zh, as soon as dW1's products of the tile before have read it (dW2's are still under way)
            if (!(ok = umma_wait(&sh.z_empty, (t & 1) ^ 1, &sh.abort))) break;
            if (t > 0 && !(ok = umma_wait(&sh.pre_full, (t - 1) & 1, &sh.abort))) break;  // and its own (another lane's, which no order binds to those)
            // (every warp writes the same bytes, and reads its own)
#pragma unroll
            for (int i = 0; i < kWords; ++i) reinterpret_cast<unsigned *>(sh.exponents)[i * 32 + lane] = exps[i];
            __syncwarp();
            const int lane0 = worked_out_here(lane);
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int q = i * 32 + lane0, row = q * per_unit >> 16, u = q - row * units;
                if (row >= 32) continue;
                const int e = sh.exponents[(first + row) * groups + u / 2];
                const int d = e - largest + 8;  // (e of a group that is not finite lies above)
                const __half s = e == 255 ? __ushort_as_half(0x7e00) : d < -24 ? __ushort_as_half(0) : __float2half_rn(power_of_two(d));
                uint4 lo, hi;
                decode_codes(code[i], __half2half2(s), lo, hi);
                uint8_t *to = zt + (u / 4) * kCkTile;
                const int k = 16 * (u % 4);
                *reinterpret_cast<uint4 *>(to + half_place(first + row, k)) = lo;
                *reinterpret_cast<uint4 *>(to + half_place(first + row, k + 8)) = hi;
            }
            // dy: the largest of the tile from the four of them (the sums over its rows want one unit, and dh is as good in it)
            const float2 own = reinterpret_cast<const float2 *>(sh.dy_units)[rows.column(lane)];
            const unsigned mine = rows.largest(own);
            if (lane == 0) {
                sh.dy_most[t & 1][warp - kCkProducer0] = mine;
                mbar_arrive(&sh.dy_known);
            }
            if (!(ok = umma_wait(&sh.dy_known, t & 1, &sh.abort))) break;
            unsigned field = 0;
#pragma unroll
            for (int q = 0; q < kCkProducers; ++q) field = max(field, sh.dy_most[t & 1][q]);
            field = max(row_unit(field), (unsigned)sh.least_field);
            if (!(ok = umma_wait(&sh.dy_empty, (t & 1) ^ 1, &sh.abort))) break;
            rows.store(dyt, dyt + kCkTile, make_float2(from_row_unit(field) * own.x, from_row_unit(field) * own.y), first, lane);
            sh.mask[0][first + lane] = mask.x;
            sh.mask[1][first + lane] = mask.y;
            sh.mask[2][first + lane] = mask.z;
            sh.mask[3][first + lane] = mask.w;
            if (warp == kCkProducer0 && lane == 0) {
                sh.z_unit = largest - 133 - 8;
                sh.dy_unit = (int)field - 127;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.op_full);
                if (issues) ok = before(t);
            }
            ok = __shfl_sync(kFull, (int)ok, 0) != 0;
            if (t + 1 < ntile) load(t + 1);
        }
        if (!ok && lane == 0) {
            atomicOr(a.status, issues ? CK_STATUS_MMA : CK_STATUS_PRODUCER);
            __nanosleep(20000);  // copies in flight land before the CTA leaves
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2;  // hidden units 32 quarter + lane, rows 64 half .. + 63 of a tile
        const unsigned tlane = tmem + ((unsigned)(quarter * 32) << 16);
        const int unit1 = head.hidden1[quarter * 32 + lane], unit2 = head.hidden2[quarter * 32 + lane];
        const float bias = __ldg(a.b1 + quarter * 32 + lane);
        if (warp == 0) {
            const bool settle = ck_apart(a, header, column, further, group);
            if (lane == 0) {
                sh.settle = settle;
                sh.add1 = sh.most1 = w1;
                sh.add2 = w2_unit;
            }
        }
        ck_epilogue_barrier();
        if (sh.settle) ck_settle(sh, a, base, ntile);
        if (lane == 0) mbar_arrive(&sh.units);
        const int add1 = sh.add1, most1 = sh.most1, add2 = sh.add2;
        sh.back[half][quarter * 32 + lane] = make_float2(channel_factor(unit2), channel_factor(unit1));  // of a hidden unit's dW1 and dW2
        const float b1 = bias * power_of_two(-unit1);
        const int b1_unit = b1 > 0.f && finite_magnitude(b1) ? binade(finite_magnitude(b1)) : -1000;  // (below zero it makes h smaller)
        // a lane of the first warp issues the sums over the rows: it knows first that their operands are there
        auto sums_of_w1 = [&](int t) -> bool {
            if (!umma_wait(&sh.dh_ready, t & 1, &sh.abort)) return false;  // which also says that tile t - 1 has left its accumulators
            tc_fence_after();
            const unsigned dh = tmem + kCkDhCol, g1 = tmem + kCkW1Col, id1 = f16_idesc((a.in + 15) / 16 * 16, true), z0 = smem_u32(zt);
            for (int ks = 0; ks < 8; ++ks) umma_f16_ts(g1, dh + 16 * ks + 8, umma_desc_rows(z0 + 2048 * ks, kCkTile), id1, ks != 0);
            for (int ks = 0; ks < 8; ++ks) umma_f16_ts(g1, dh + 16 * ks, umma_desc_rows(z0 + 2048 * ks, kCkTile), id1, 1);
            umma_commit(&sh.z_empty);
            umma_commit(&sh.g1_full);
            return true;
        };
        auto sums_of_w2 = [&](int t) -> bool {
            if (!umma_wait(&sh.pre_ready, t & 1, &sh.abort)) return false;
            tc_fence_after();
            const unsigned pre = tmem + kCkPreCol, g2 = tmem + kCkW2Col, id2 = f16_idesc((a.out + 15) / 16 * 16, true), dy0 = smem_u32(dyt);
            for (int ks = 0; ks < 8; ++ks) {
                umma_f16_ts(g2, pre + 16 * ks + 8, umma_desc_rows(dy0 + 2048 * ks, kCkTile), id2, ks != 0);
                umma_f16_ts(g2, pre + 16 * ks, umma_desc_rows(dy0 + kCkTile + 2048 * ks, kCkTile), id2, 1);
            }
            for (int ks = 0; ks < 8; ++ks) umma_f16_ts(g2, pre + 16 * ks, umma_desc_rows(dy0 + 2048 * ks, kCkTile), id2, 1);
            umma_commit(&sh.dy_empty);
            umma_commit(&sh.g2_full);
            return true;
        };
        const int nb1 = (a.in + 15) / 16, nb = nb1 + (a.out + 15) / 16;
        float sums[kBlocks][16], db = 0.f;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[b][j] = 0.f;
#pragma unroll 1
        for (int t = 0; t < ntile; ++t) {
            if (!(ok = umma_wait(&sh.dh_full, t & 1, &sh.abort, kUmmaWaitNs, 50))) break;
            tc_fence_after();
            const unsigned bit = 1u << lane;
            // masks rows 64 half .. + 63 of an accumulator (lane = hidden unit) and takes them apart
            auto apart = [&](unsigned at, auto value) {
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int row = 64 * half + 16 * c;
                    unsigned r[16], parts[16];
                    tmem_ld16(at + row, r);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const uint4 m = *reinterpret_cast<const uint4 *>(&sh.mask[quarter][row + j]);
                        const unsigned mw[4] = {m.x, m.y, m.z, m.w};
                        float v[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) v[q] = value(__uint_as_float(r[j + q]), (mw[q] & bit) != 0, q);
                        split_halves(v[0], v[1], parts[j / 2], parts[8 + j / 2]);
                        split_halves(v[2], v[3], parts[j / 2 + 1], parts[8 + j / 2 + 1]);
                    }
                    tmem_st16(at + row, parts);
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
            };
            float partial[4] = {};
            apart(tlane + kCkDhCol, [&](float v, bool alive, int q) {
                v = alive ? v * kDhUnit : 0.f;
                partial[q] += v;
                return v;
            });
            if (lane == 0) {
                mbar_arrive(&sh.dh_ready);
                if (warp == 0) ok = sums_of_w1(t);
            }
            __syncwarp();
            // units: zh 2^zu, W1 2^(w1 - 14); h in units of 2^hu, which the largest sum (176 x 2^15 x 32512 in the accumulator's) and bias leave
            // below 1.2 x 2^15
            const int dyu = sh.dy_unit, zu = sh.z_unit, hu = max(zu + most1 + 24, b1_unit + 2) - 15;
            const float to_h = power_of_two(max(zu + add1 - kOperand - hu, -126)), shift = b1 * power_of_two(min(max(-hu, -126), 127));
            if (!umma_wait(&sh.pre_full, t & 1, &sh.abort, kUmmaWaitNs, 50)) ok = false;
            tc_fence_after();
            apart(tlane + kCkPreCol, [&](float v, bool alive, int) { return alive ? __fmaf_rn(v, to_h, shift) : 0.f; });
            if (lane == 0) {
                mbar_arrive(&sh.pre_ready);
                if (warp == 0) ok = ok && sums_of_w2(t);
            }
            if (!(ok = __shfl_sync(kFull, (int)ok, 0) != 0)) break;
            // what the tile's sums are multiples of: products of powers of two, zero below the smallest number (sums below 2^-112 may be lost)
            auto scale = [](int e) { return power_of_two(max(min(e, 127), -126)) * power_of_two(max(min(e + 126, 0), -126)); };
            db += (partial[0] + partial[1] + (partial[2] + partial[3])) * scale(dyu + add2);
            if (!(ok = umma_wait(&sh.g1_full, t & 1, &sh.abort, kUmmaWaitNs, 50))) break;
            tc_fence_after();
            bool both = false;  // dW2's sums are there as well
            const float f1 = scale(dyu + add2 + zu), f2 = scale(dyu - kOperand + hu);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                const int b = 2 * i + half;
                if (b >= nb) break;
                if (b >= nb1 && !both) {
                    if (!(ok = umma_wait(&sh.g2_full, t & 1, &sh.abort, kUmmaWaitNs, 50))) break;
                    tc_fence_after();
                    both = true;
                }
                unsigned r[16];
                tmem_ld16(tlane + (b < nb1 ? kCkW1Col + 16 * b : kCkW2Col + 16 * (b - nb1)), r);
                tc_wait_ld();
                const float f = b < nb1 ? f1 : f2;
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[i][j] = __fmaf_rn(__uint_as_float(r[j]), f, sums[i][j]);
            }
            tc_fence_before();
            if (!ok) break;
        }
        if (!ok && lane == 0) atomicOr(a.status, CK_STATUS_EPILOGUE);
        // db1 in column `in`: both halves of the rows through shared memory.  (A warp that gave up comes here as well: the barriers want all.)
        const float f1 = sh.back[half][quarter * 32 + lane].x, f2 = sh.back[half][quarter * 32 + lane].y;
        db *= f1;
        float *prow = a.partial + ((long long)blockIdx.x * 128 + quarter * 32 + lane) * (a.N1p + a.N2p);
        if (half == 1) sh.both[quarter * 32 + lane] = db;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const int b = 2 * i + half;
            if (b >= nb) break;
            float *to = prow + (b < nb1 ? 16 * b : a.N1p + 16 * (b - nb1));
            const float f = b < nb1 ? f1 * sh.z_back[b / 2] : f2, *back = b < nb1 ? nullptr : sh.dy_back + 16 * (b - nb1);
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[i][j] *= back ? f * back[j] : f;
#pragma unroll
            for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4 *>(to + j) = make_float4(sums[i][j], sums[i][j + 1], sums[i][j + 2], sums[i][j + 3]);
        }
        ck_epilogue_barrier();  // (column `in` may lie in a block of the other half)
        if (half == 0) prow[a.in] = db + sh.both[quarter * 32 + lane];
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kCkProducer0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- forward -----------------------------------------------------------------------------------------------------------
//     y = relu(z W1^T + b1) W2^T, leaving codes and exponents of z and the bits of the ReLU
//
// Tiles of 128 rows again, lane = row from the first product on.  Sixteen producer warps hold eight rows each, two columns a lane: the
// maxima of the groups give the exponents, those of the rows their units; codes leave, heads and tails go to a ring of two slots of 64
// columns.  The products with a tail have an accumulator of their own (an addition to a sum cuts off what lies below its last bit: 11
// additions at 163 inputs instead of 33), which four epilogue warps add; h goes back in heads and tails in place, in units that no row
// can exceed: with z in units of its row, W1 of its matrix and the largest bias known, a bound is at hand, and 2^-25 below it is float16's
// smallest tail.  The second layer's sums take the place of the products with tails.
constexpr int kFwProducers = 16, kFwThreads = 20 * 32;  // (twenty warps: 96 registers a thread; one more would cost 16 of them)
constexpr int kFwSlot = 2 * kCkTile, kFwSlots = 2;
struct CkForwardShared {
    uint64_t image, slot_full[kFwSlots], slot_empty[kFwSlots], h_full[2], h_ready[2], y_full[2], y_read[2], y_written, y_copied;
    alignas(16) float b1[128];
    int units[4][kCkRows];
    unsigned z_groups[8];  // the largest exponent of each group in this CTA's rows
    float outputs[64], hidden[128];  // units of W2's columns, and what a hidden unit weighs against the largest
    uint32_t tmem_base;
    int abort;
};
struct CkForwardArgs {
    const float *z, *b1;
    const uint8_t *image;
    float *y;
    int8_t *codes;
    uint8_t *exponents;
    uint2 *mask;          // [rows][2]
    uint8_t *z_groups;    // [ctas][8]
    long long rows;
    int in, out, pitch, chunks, tiles;
    unsigned *status;
};
static int ck_forward_smem(int chunks, int out) { return 1024 + (2 * chunks + 2) * kCkTile + kFwSlots * kFwSlot + kCkRows * out * 4 + 16; }

template <int kChunks>
__global__ void __launch_bounds__(kFwThreads, 1) mlp_checkpoint_forward_kernel(const __grid_constant__ CkForwardArgs a) {
    after_previous_kernel();
    extern __shared__ uint8_t ck_raw[];
    __shared__ CkForwardShared sh;
    uint8_t *base = ck_raw + ((1024u - (smem_u32(ck_raw) & 1023u)) & 1023u);
    uint8_t *w2 = base + 2 * kChunks * kCkTile, *ring = w2 + 2 * kCkTile;
    float *ytile = reinterpret_cast<float *>(ring + kFwSlots * kFwSlot);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&sh.image, 1);
        for (int q = 0; q < kFwSlots; ++q) {
            mbar_init(&sh.slot_full[q], kFwProducers);
            mbar_init(&sh.slot_empty[q], 1);
        }
        for (int q = 0; q < 2; ++q) {
            mbar_init(&sh.h_full[q], 2);  // the products, and the MMA lane itself: what it has seen of the units the epilogue sees
            mbar_init(&sh.h_ready[q], 4);
            mbar_init(&sh.y_full[q], 1);
            mbar_init(&sh.y_read[q], 4);
        }
        mbar_init(&sh.y_written, 4);
        mbar_init(&sh.y_copied, 4);
        sh.abort = 0;
        mbar_fence_init();
    }
    const CkHeader &head = *reinterpret_cast<const CkHeader *>(a.image);
    const int apart = head.apart;
    if (threadIdx.x < 128) sh.b1[threadIdx.x] = __ldg(a.b1 + threadIdx.x) * power_of_two(-head.hidden1[threadIdx.x]);
    if (threadIdx.x < 8) sh.z_groups[threadIdx.x] = 0;
    if (warp == kFwProducers) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = sh.tmem_base;  // h of two tiles at 0 and 128, what goes with tails (then y) at 256 and 384
    const int ntile = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    auto row_of = [&](int it) { return ((long long)blockIdx.x + (long long)it * gridDim.x) * kCkRows; };
    bool ok = true;

    if (warp < kFwProducers) {
        const int first = warp * 8, groups = (a.in + 31) / 32;
        // place of (row r, columns 2 lane, 2 lane + 1) in a slot: units of eight columns change places by the row's lowest three bits
        const int word = (lane & 3) * 4;
        int s = 0;
        unsigned ph = 1, groups_most = 0;  // a byte for each chunk: group 2 c + lane / 16
#pragma unroll 1
        for (int t = 0; t < ntile && ok; ++t) {
            const long long row0 = row_of(t) + first;
            float2 v[8][kChunks];
            {
                const int k = 64 * (kChunks - 1) + 2 * lane, in = worked_out_here(a.in);
                const bool one = k < a.in, two = k + 1 < a.in;
                const float *p0 = a.z + (row0 < a.rows ? row0 : a.rows - 1) * a.in + 2 * lane;
                const int last = (int)(a.rows - 1 - row0 < 7 ? max((int)(a.rows - 1 - row0), 0) : 7);
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float *p = p0 + min(r, last) * in;  // (a row that does not exist is read as the last one: nothing of it leaves)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        v[r][c].x = c + 1 < kChunks || one ? __ldg(p + 64 * c) : 0.f;
                        v[r][c].y = c + 1 < kChunks || two ? __ldg(p + 64 * c + 1) : 0.f;
                    }
                }
            }
            // codes are put together in this warp's rows of the slot that the first chunk is going to: five rows where its heads will be,
            // three where its tails (in two bytes a lane they would go to memory in pieces of sectors, which cost 13,000 clocks a tile)
            if (!(ok = umma_wait(&sh.slot_empty[s], ph, &sh.abort))) break;
            uint8_t *const low = ring + s * kFwSlot + first * 128, *const high = low + kCkTile;
            unsigned own = 0;  // the largest finite magnitude of row (lane & 15) / 2, as far as seen
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                unsigned m[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) m[r] = max(magnitude(v[r][c].x), magnitude(v[r][c].y));
                const unsigned most = gather_max8<16>(m);  // of row (lane & 15) / 2 and the 32 columns of this half of the warp
                const bool finite = most < 0x7f800000u;
                const unsigned e = rows8_exponent(most);
                const float to_units = rows8_to_units(e);
                const int r8 = (lane & 15) >> 1, g = 2 * c + (lane >> 4);
                if ((lane & 1) == 0 && g < groups) high[768 + r8 * groups + g] = (uint8_t)e;
                groups_most = __vmaxu4(groups_most, (finite && e > 7u ? e : 0u) << (8 * c));  // (7: nothing but zeros, or next to it)
                unsigned f = finite ? most : 0u;
                if (__any_sync(kFull, !finite)) {  // what is finite of such groups, for the unit of the row
#pragma unroll
                    for (int r = 0; r < 8; ++r) m[r] = max(finite_magnitude(v[r][c].x), finite_magnitude(v[r][c].y));
                    f = gather_max8<16>(m);
                }
                own = max(own, max(f, __shfl_xor_sync(kFull, f, 16)));
                const int k = 64 * c + 2 * lane, pitch = worked_out_here(a.pitch);
                auto put = [&](auto clamp) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const float u = __shfl_sync(kFull, to_units, max8_lane<16>(r));
                        unsigned x = __float_as_uint(__fmaf_rn(v[r][c].x, u, kRoundWhole)), y = __float_as_uint(__fmaf_rn(v[r][c].y, u, kRoundWhole));
                        if constexpr (decltype(clamp)::value) {
                            x = (unsigned)rows8_code(v[r][c].x, u);
                            y = (unsigned)rows8_code(v[r][c].y, u);
                        }
                        if (k < pitch) *reinterpret_cast<uint16_t *>((r < 5 ? low + r * pitch : high + (r - 5) * pitch) + k) = (uint16_t)__byte_perm(x, y, 0x0040);
                    }
                };
                if (__any_sync(kFull, e >= 254u)) put(std::true_type());  // up to 128 units in the last binade, or groups that are not finite
                else put(std::false_type());
            }
            __syncwarp();
            {
                const int in_low = 5 * a.pitch / 16, total = 8 * a.pitch / 16;
                const long long left = (a.rows - row0) * a.pitch / 16;  // (may be <= 0)
                for (int q = lane; q < total && q < left; q += 32)
                    reinterpret_cast<uint4 *>(a.codes + row0 * a.pitch)[q] = *reinterpret_cast<const uint4 *>(q < in_low ? low + 16 * q : high + 16 * (q - in_low));
                if (row0 + 8 <= a.rows) {
                    if (lane < groups) reinterpret_cast<uint2 *>(a.exponents + row0 * groups)[lane] = *reinterpret_cast<const uint2 *>(high + 768 + 8 * lane);
                } else {
                    for (int q = lane; q < 8 * groups; q += 32)
                        if (row0 + q / groups < a.rows) a.exponents[row0 * groups + q] = high[768 + q];
                }
            }
            __syncwarp();
            if (apart & CK_INPUTS) {  // in units of W1's columns, of which the row's largest is another
                unsigned m[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    m[r] = 0;
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        const float2 f = make_float2(channel_factor(head.inputs[64 * c + 2 * lane]), channel_factor(head.inputs[64 * c + 2 * lane + 1]));
                        v[r][c].x *= f.x;
                        v[r][c].y *= f.y;
                        m[r] = max(m[r], max(finite_magnitude(v[r][c].x), finite_magnitude(v[r][c].y)));
                    }
                }
                own = __shfl_sync(kFull, gather_max8(m), 4 * ((lane & 15) >> 1));
            }
            const unsigned field = row_unit(own);
            if (lane < 16 && (lane & 1) == 0) sh.units[t & 3][first + (lane >> 1)] = (int)field - 127;
            const float scale = from_row_unit(field);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float u = __shfl_sync(kFull, scale, 2 * r);
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    unsigned head, tail;
                    split_halves(v[r][c].x * u, v[r][c].y * u, head, tail);
                    v[r][c] = make_float2(__uint_as_float(head), __uint_as_float(tail));
                }
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                if (c > 0 && !(ok = umma_wait(&sh.slot_empty[s], ph, &sh.abort))) break;
                uint8_t *to = ring + s * kFwSlot + first * 128 + word;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int at = r * 128 + (((lane >> 2) ^ r) << 4);
                    *reinterpret_cast<float *>(to + at) = v[r][c].x;
                    *reinterpret_cast<float *>(to + kCkTile + at) = v[r][c].y;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.slot_full[s]);
                if (++s == kFwSlots) {
                    s = 0;
                    ph ^= 1;
                }
            }
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) groups_most = __vmaxu4(groups_most, __shfl_xor_sync(kFull, groups_most, d));
        if ((lane & 15) < kChunks) atomicMax(&sh.z_groups[2 * (lane & 15) + (lane >> 4)], groups_most >> (8 * (lane & 15)) & 0xffu);
        if (!ok && lane == 0) atomicOr(a.status, CK_STATUS_PRODUCER);
    } else {
        const int quarter = warp & 3, row = quarter * 32 + lane;
        if (quarter == 0 && lane == 0) ck_copy_image(base, a.image, kChunks, &sh.image);
        if (apart & (CK_OUTPUTS | CK_HIDDEN)) {
            if (row < 64) sh.outputs[row] = channel_factor(head.outputs[row]);
            sh.hidden[row] = channel_factor(head.hidden1[row] + head.hidden2[row] - head.hidden);
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (apart & CK_HIDDEN) {  // W2 with what its hidden unit weighs in y
                umma_wait(&sh.image, 0, &sh.abort);
                ck_rescale(w2, w2 + kCkTile, 1, sh.hidden, nullptr, 128);
                fence_proxy_async();
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
        }
        // a lane of the first warp issues the MMAs as well: while the producers fill the slots there is little else for it to do
        const bool issues = quarter == 0;
        auto first_layer = [&](int t) -> bool {
            const int b = t & 1, steps = (a.in + 15) / 16;
            const unsigned id1 = f16_idesc(128, false);
            const uint64_t w1h = umma_desc(smem_u32(base)), w1l = umma_desc(smem_u32(base + kChunks * kCkTile));
            if (t == 0 && !umma_wait(&sh.image, 0, &sh.abort)) return false;
            if (!umma_wait(&sh.y_read[b], ((t >> 1) & 1) ^ 1, &sh.abort)) return false;  // y of tile t - 2: nothing of it is left
            tc_fence_after();
            const unsigned d = tmem + 128 * b, small = tmem + 256 + 128 * b;
            int q = t * kChunks;
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c, ++q) {
                const int s = q % kFwSlots;
                if (!umma_wait(&sh.slot_full[s], (q / kFwSlots) & 1, &sh.abort)) return false;
                tc_fence_after();
                const uint64_t zh = umma_desc(smem_u32(ring + s * kFwSlot)), zl = umma_desc(smem_u32(ring + s * kFwSlot + kCkTile));
                const uint64_t wh = w1h + (uint64_t)(c * (kCkTile >> 4)), wl = w1l + (uint64_t)(c * (kCkTile >> 4));
                const int here = min(4, steps - 4 * c);
                for (int ks = 0; ks < here; ++ks) {
                    umma_f16(small, zl + 2 * ks, wh + 2 * ks, id1, (c | ks) != 0);
                    umma_f16(small, zh + 2 * ks, wl + 2 * ks, id1, 1);
                }
                for (int ks = 0; ks < here; ++ks) umma_f16(d, zh + 2 * ks, wh + 2 * ks, id1, (c | ks) != 0);
                umma_commit(&sh.slot_empty[s]);
            }
            umma_commit(&sh.h_full[b]);
            mbar_arrive(&sh.h_full[b]);
            return true;
        };
        auto second_layer = [&](int t) -> bool {
            const int b = t & 1;
            const unsigned id2 = f16_idesc((a.out + 15) / 16 * 16, true), w2h = smem_u32(w2), w2l = smem_u32(w2 + kCkTile);
            if (!umma_wait(&sh.h_ready[b], (t >> 1) & 1, &sh.abort)) return false;
            tc_fence_after();
            const unsigned d = tmem + 256 + 128 * b, ah = tmem + 128 * b;
            for (int ks = 0; ks < 8; ++ks) {
                umma_f16_ts(d, ah + 16 * ks + 8, umma_desc_rows(w2h + 2048 * ks, kCkTile), id2, ks != 0);
                umma_f16_ts(d, ah + 16 * ks, umma_desc_rows(w2l + 2048 * ks, kCkTile), id2, 1);
            }
            for (int ks = 0; ks < 8; ++ks) umma_f16_ts(d, ah + 16 * ks, umma_desc_rows(w2h + 2048 * ks, kCkTile), id2, 1);
            umma_commit(&sh.y_full[b]);
            return true;
        };
        auto issue = [&](bool did) {  // what lane 0 says goes for the warp
            did = __shfl_sync(kFull, (int)did, 0) != 0;
            return did;
        };
        const unsigned tlane = tmem + ((unsigned)(quarter * 32) << 16);
        const int w1 = head.w1, b1_unit = head.b1, w2_unit = head.w2 + head.hidden - kOperand;
        // h is below 2^(zr + w1 + 10) by its products (176 of numbers below two units each) and 2^(b1 + 1) by its bias: twice 2^14 of its units
        auto unit_of = [&](int t) { return max(sh.units[t & 3][row] + w1 + 10, b1_unit + 1) - 14; };
        auto leave = [&](int t) -> bool {  // y of tile t
            const int b = t & 1;
            const long long row0 = row_of(t);
            const int e = unit_of(t) + w2_unit, e1 = max(min(e, 127), -126);
            const float unit = power_of_two(e1), rest = power_of_two(max(e - e1, -126));
            if (!umma_wait(&sh.y_copied, (t & 1) ^ 1, &sh.abort)) return false;
            if (!umma_wait(&sh.y_full[b], (t >> 1) & 1, &sh.abort)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < a.out; c0 += 16) {
                unsigned r[16];
                tmem_ld16(tlane + 256 + 128 * b + c0, r);
                tc_wait_ld();
                float y[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = __uint_as_float(r[j]) * unit * rest;
                if (apart & CK_OUTPUTS) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) y[j] *= sh.outputs[c0 + j];
                }
                put_16(ytile + row * a.out + c0, a.out - c0, a.out, lane, y);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.y_read[b]);
                mbar_arrive(&sh.y_written);
            }
            if (!umma_wait(&sh.y_written, t & 1, &sh.abort)) return false;
            const int here = a.rows - row0 < kCkRows ? (int)(a.rows - row0) : kCkRows, total = here * a.out;
            float *out = a.y + row0 * a.out;  // (128 rows of any width are a multiple of 16 bytes)
            const int quads = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 ? total / 4 : 0;
            for (int q = row; q < quads; q += 128) reinterpret_cast<float4 *>(out)[q] = reinterpret_cast<const float4 *>(ytile)[q];
            for (int q = 4 * quads + row; q < total; q += 128) out[q] = ytile[q];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.y_copied);
            return true;
        };
#pragma unroll 1
        for (int t = 0; t < ntile; ++t) {
            const int b = t & 1;
            if (issues && !(ok = issue(lane != 0 || first_layer(t)))) break;
            if (!(ok = umma_wait(&sh.h_full[b], (t >> 1) & 1, &sh.abort))) break;
            tc_fence_after();
            const int hu = unit_of(t);
            const float f1 = power_of_two(max(sh.units[t & 3][row] + w1 - 2 * kOperand - hu, -126)), f2 = power_of_two(min(max(-hu, -126), 127));
            unsigned bits[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) bits[w] = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    const int c0 = 32 * w + 16 * half;
                    unsigned r[16], q[16], parts[16], word = 0;
                    tmem_ld16(tlane + 128 * b + c0, r);
                    tmem_ld16(tlane + 256 + 128 * b + c0, q);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 bias = *reinterpret_cast<const float4 *>(&sh.b1[c0 + j]);
                        const float bw[4] = {bias.x, bias.y, bias.z, bias.w};
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[i] = fmaxf(__fmaf_rn(__uint_as_float(r[j + i]) + __uint_as_float(q[j + i]), f1, bw[i] * f2), 0.f);
                            word |= v[i] > 0.f ? 1u << (j + i) : 0u;
                        }
                        split_halves(v[0], v[1], parts[j / 2], parts[8 + j / 2]);
                        split_halves(v[2], v[3], parts[j / 2 + 1], parts[8 + j / 2 + 1]);
                    }
                    bits[w] |= word << (16 * half);
                    tmem_st16(tlane + 128 * b + c0, parts);
                }
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.h_ready[b]);
            if (issues && !(ok = issue(lane != 0 || second_layer(t)))) break;
            const long long at = row_of(t) + row;
            if (at < a.rows) reinterpret_cast<uint4 *>(a.mask)[at] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
            if (t > 0 && !(ok = leave(t - 1))) break;
        }
        if (ok && ntile > 0) ok = leave(ntile - 1);
        if (!ok && issues && lane == 0) __nanosleep(20000);  // copies in flight land before the CTA leaves
        if (!ok && lane == 0) atomicOr(a.status, CK_STATUS_EPILOGUE);
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < 8) a.z_groups[blockIdx.x * 8 + threadIdx.x] = (uint8_t)sh.z_groups[threadIdx.x];
    if (warp == kFwProducers) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
// header | matrices | what the forward saw of its CTAs' rows: the largest exponent of each group of z
static int64_t ck_matrices_end(int in_dim) { return kCkHeader + (int64_t)(2 * ((in_dim + 63) / 64) + 2) * kCkTile; }
static int64_t ck_image_bytes(int in_dim) { return ck_matrices_end(in_dim) + 148 * 8; }
static GradReduce ck_reduce(int64_t rows, int in_dim, int out_dim) {
    GradReduce r = {};
    const int64_t tiles = (rows + kCkRows - 1) / kCkRows;
    r.in_dim = in_dim; r.out_dim = out_dim; r.N1p = grad_round16(in_dim + 1); r.N2p = grad_round16(out_dim);
    r.ctas = (int)(tiles < 148 ? tiles : 148);
    return r;
}
static int64_t ck_partial_floats(const GradReduce &r) { return (int64_t)r.ctas * kCkRows * (r.N1p + r.N2p); }
static int64_t ck_column_words(const GradReduce &r) { return (int64_t)r.ctas * kCkProducers * 64; }

template <typename Kernel>
static int ck_launch(Kernel kernel, const char *name, const CkArgs &a, int smem, int ctas, cudaStream_t st) {
    int unused = 0;  // raises the kernel's limit of shared memory on this device
    const int rc = persistent_ctas(kernel, kCkThreads, (size_t)smem, &unused);
    if (rc != NPA_OK) return rc;
    launch_early(kernel, ctas, kCkThreads, (size_t)smem, st, a);
    return check_launch(name);
}

int check_mlp8(const char *me, int64_t rows, int32_t in_dim, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || out_dim <= 0) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: rows, in_dim and out_dim must be positive", me);
    if (rows > ((int64_t)1 << 31) - 1 || in_dim > kCkMaxIn || out_dim > kCkMaxOut)
        return fail(NPA_ERR_UNSUPPORTED, "%s: supports fewer than 2^31 rows, in <= %d and out <= %d (hidden width 128), got %lld, %d and %d", me, kCkMaxIn,
                    kCkMaxOut, (long long)rows, in_dim, out_dim);
    return NPA_OK;
}

}  // namespace npa

using namespace npa;

extern "C" {

int64_t npa_mlp_checkpoint_image_bytes(int32_t in_dim) { return in_dim <= 0 ? 0 : ck_image_bytes(in_dim); }

int npa_mlp_checkpoint_forward(const float *z, const float *W1, const float *b1, const float *W2, float *y, int64_t rows, int32_t in_dim, int32_t out_dim,
                               int64_t w1_stride_out, int64_t w1_stride_in, int64_t w2_stride_out, int64_t w2_stride_in, void *codes, uint8_t *exponents,
                               uint32_t *mask, void *image, int64_t image_bytes, void *stream) {
    const char *me = "npa_mlp_checkpoint_forward";
    int rc = check_mlp8(me, rows, in_dim, out_dim);
    if (rc != NPA_OK) return rc;
    if (!z || !W1 || !b1 || !W2 || !y || !codes || !exponents || !mask) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be non-NULL", me);
    if (!image || ((uintptr_t)image | (uintptr_t)codes | (uintptr_t)mask | (uintptr_t)exponents) % 16)
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: codes, exponents, mask and image must be there, 16-byte aligned", me);
    if (((uintptr_t)z | (uintptr_t)W1 | (uintptr_t)b1 | (uintptr_t)W2 | (uintptr_t)y) % 4) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every array must be float aligned", me);
    const int64_t need = ck_image_bytes(in_dim);
    if (image_bytes < need) return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: image has %lld bytes, %lld needed", me, (long long)image_bytes, (long long)need);
    CkForwardArgs a = {};
    a.z = z; a.b1 = b1; a.image = static_cast<const uint8_t *>(image); a.y = y; a.codes = static_cast<int8_t *>(codes); a.exponents = exponents;
    a.mask = reinterpret_cast<uint2 *>(mask); a.z_groups = static_cast<uint8_t *>(image) + ck_matrices_end(in_dim); a.rows = rows; a.in = in_dim; a.out = out_dim; a.pitch = (int)rows8_pitch(in_dim);
    a.chunks = (in_dim + 63) / 64; a.tiles = (int)((rows + kCkRows - 1) / kCkRows);
    if (!(a.status = umma_status_word())) return fail(NPA_ERR_CUDA, "%s: no status word", me);
    const cudaStream_t st = (cudaStream_t)stream;
    const CkImageArgs make{W1, b1, W2, w1_stride_out, w1_stride_in, w2_stride_out, w2_stride_in, in_dim, out_dim, a.chunks, static_cast<uint8_t *>(image)};
    launch_early(mlp_checkpoint_image_kernel, ck_image_blocks(a.chunks), kImageThreads, 0, st, make);
    if ((rc = check_launch("mlp_checkpoint_image_kernel")) != NPA_OK) return rc;
    const auto kernel = a.chunks == 1 ? mlp_checkpoint_forward_kernel<1> : a.chunks == 2 ? mlp_checkpoint_forward_kernel<2> : mlp_checkpoint_forward_kernel<3>;
    const int smem = ck_forward_smem(a.chunks, out_dim);
    int unused = 0;  // raises the kernel's limit of shared memory on this device
    if ((rc = persistent_ctas(kernel, kFwThreads, (size_t)smem, &unused)) != NPA_OK) return rc;
    launch_early(kernel, a.tiles < 148 ? a.tiles : 148, kFwThreads, (size_t)smem, st, a);
    return check_launch("mlp_checkpoint_forward_kernel");
}

int64_t npa_mlp_checkpoint_backward_scratch_bytes(int64_t rows, int32_t in_dim, int32_t out_dim) {
    if (rows <= 0 || in_dim <= 0 || out_dim <= 0) return 0;
    const GradReduce r = ck_reduce(rows, in_dim, out_dim);
    return 4 * (ck_partial_floats(r) + ck_column_words(r));
}

int npa_mlp_checkpoint_backward(const void *codes, const uint8_t *exponents, const uint32_t *mask, const void *image, int64_t image_bytes, const float *b1,
                                const float *dy, float *dz, float *dW1, float *db1, float *dW2, int64_t rows, int32_t in_dim, int32_t out_dim, void *scratch,
                                int64_t scratch_bytes, void *stream) {
    const char *me = "npa_mlp_checkpoint_backward";
    int rc = check_mlp8(me, rows, in_dim, out_dim);
    if (rc != NPA_OK) return rc;
    if (!codes || !exponents || !mask || !image || !b1 || !dy) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: every input must be non-NULL", me);
    if ((!dW1 || !db1 || !dW2) && (dW1 || db1 || dW2)) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: dW1, db1 and dW2 come together", me);
    if (!scratch || ((uintptr_t)scratch | (uintptr_t)codes | (uintptr_t)exponents | (uintptr_t)mask | (uintptr_t)image | (uintptr_t)dy) % 16)
        return fail(NPA_ERR_INVALID_ARGUMENT, "%s: codes, exponents, mask, image, dy and scratch must be there, 16-byte aligned", me);
    if (((uintptr_t)dz | (uintptr_t)b1) % 4) return fail(NPA_ERR_INVALID_ARGUMENT, "%s: dz and b1 must be float aligned", me);
    if (image_bytes < ck_image_bytes(in_dim))
        return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: image has %lld bytes, %lld needed", me, (long long)image_bytes, (long long)ck_image_bytes(in_dim));
    const int64_t need = npa_mlp_checkpoint_backward_scratch_bytes(rows, in_dim, out_dim);
    if (scratch_bytes < need) return fail(NPA_ERR_SCRATCH_TOO_SMALL, "%s: scratch has %lld bytes, %lld needed", me, (long long)scratch_bytes, (long long)need);
    if (!dz && !dW1) return NPA_OK;
    const cudaStream_t st = (cudaStream_t)stream;
    GradReduce r = ck_reduce(rows, in_dim, out_dim);
    CkArgs a = {};
    a.codes = static_cast<const int8_t *>(codes); a.exponents = exponents; a.mask = reinterpret_cast<const uint4 *>(mask); a.dy = dy; a.b1 = b1;
    a.image = static_cast<const uint8_t *>(image); a.dz = dz; a.partial = static_cast<float *>(scratch);
    a.dy_columns = reinterpret_cast<unsigned *>(a.partial + ck_partial_floats(r)); a.looked = dz != nullptr;
    a.z_groups = a.image + ck_matrices_end(in_dim);
    a.rows = rows; a.in = in_dim; a.out = out_dim; a.pitch = (int)rows8_pitch(in_dim); a.chunks = (in_dim + 63) / 64; a.N1p = r.N1p; a.N2p = r.N2p;
    a.tiles = (int)((rows + kCkRows - 1) / kCkRows);
    if (!(a.status = umma_status_word())) return fail(NPA_ERR_CUDA, "%s: no status word", me);
    const bool two = out_dim > 32;
    const auto dz_kernel = in_dim % 4 ? (two ? mlp_checkpoint_dz_kernel<true, false> : mlp_checkpoint_dz_kernel<false, false>)
                                      : (two ? mlp_checkpoint_dz_kernel<true, true> : mlp_checkpoint_dz_kernel<false, true>);
    if (dz && (rc = ck_launch(dz_kernel, "mlp_checkpoint_dz_kernel", a, ck_dz_smem(a.chunks, in_dim), r.ctas, st)) !=
                  NPA_OK)
        return rc;
    if (!dW1) return NPA_OK;
    const bool few = (in_dim + 15) / 16 + (out_dim + 15) / 16 <= 8;
    const auto kernel = few ? (two ? mlp_checkpoint_weights_kernel<4, true> : mlp_checkpoint_weights_kernel<4, false>)
                            : (two ? mlp_checkpoint_weights_kernel<7, true> : mlp_checkpoint_weights_kernel<7, false>);
    if ((rc = ck_launch(kernel, "mlp_checkpoint_weights_kernel", a, ck_weights_smem(a.chunks), r.ctas, st)) != NPA_OK) return rc;
    r.partial = a.partial; r.dW1 = dW1; r.dW2 = dW2; r.db1 = db1;
    return launch_grad_reduce(r, st);
}

}  // extern "C"
