// Rows of bytes through TMA and kind::i8 MMAs: what the tensor-core kernels on 8-bit codes share (int8_tcgen05.cu, int8_mlp.cu).
#pragma once
#include <cuda.h>

#include "umma.cuh"

namespace npa {

constexpr int kI8Chunk = 128;  // bytes of K in a stage: one row of the 128-byte swizzle

enum { INT8_STATUS_LOAD = 128, INT8_STATUS_MMA = 256, INT8_STATUS_EPILOGUE = 512 };

unsigned *umma_status_word();  // mlp_tcgen05.cu
// int8_tcgen05.cu: rows of bytes as TMA reads them, boxes of 128 bytes of `box_rows` rows, 128-byte swizzle, zeros outside.
int byte_rows_map(const char *me, CUtensorMap *map, const void *p, long long pitch, long long rows, int cols, int box_rows);

__device__ inline void umma_i8(unsigned d_tmem, uint64_t a_desc, uint64_t b_desc, unsigned idesc, int accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// A box of a two-dimensional array into this CTA's shared memory; x in elements along the rows.
__device__ inline void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)), "l"(map),
                 "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}

// Instruction descriptor: M = 128, signed 8-bit x signed 8-bit -> 32-bit integers, both operands K-major.
__device__ constexpr unsigned i8_idesc(int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(128 >> 4) << 24); }

}  // namespace npa
