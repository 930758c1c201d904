// A tile of a page pool held in 8 bits: K and V of 16 tokens of one kv head with their two scales, and the codes' arithmetic.
//
// The codes lie in the order in which mma.sync m16n8k16 wants its B operand, so that a lane of the attention kernel fetches what it multiplies
// with 16-byte loads that follow one another over the lanes: no swizzle, no ldmatrix, no transposition of V. With lane = 4 g + t:
//   K, scores = Q K^T (n = token, k = dim): column c of score tile j is token 4 (c / 2) + 2 j + c % 2, and the four k elements of a lane in step s
//      are the neighbours 16 s + 4 t ..+3 (the query's fragments follow the same order). Word (s, j) of lane (g, t), the four codes of token
//      4 (g / 2) + 2 j + g % 2, is word u = 2 s + j of the lane;
//   V, output = P V (n = dim, k = token): a lane's scores of the two tiles are those of tokens 4 t ..+3, which makes them its A fragment of P
//      as they are; word i of lane (g, t) holds the codes of those tokens for dim 8 i + g.
// Codes are e4m3 numbers, or integers c kept as c + 128.
// Word u of a lane lies at 16 (32 (u / 4) + lane) + 4 (u % 4); V follows K, and behind both lie the f32 scales of K and of V and 8 bytes of nothing.
#pragma once

#include "device_utils.cuh"

#include <cuda_fp8.h>

namespace llaisys::kernels {

constexpr int kQuantTokens = 16;           // tokens of a block
constexpr float kQuantFloor = 0x1p-100f;   // smallest scale an append writes

__host__ __device__ __forceinline__ int quant_scales_at(int d) { return 2 * kQuantTokens * d; }

// Where a token lives. False (and flagged): not in the pool.
__device__ __forceinline__ bool quant_tile_of(const QuantView &kv, int seq, int block, int32_t *error_flag, unsigned char *&tiles) {
    const int in_table = block / kv.blocks_per_page;
    if (seq < 0 || seq >= kv.table_rows) {
        atomicOr(error_flag, kErrBadSeq);
        return false;
    }
    if (block < 0 || in_table >= kv.table_stride) {
        atomicOr(error_flag, kErrBadPosition);
        return false;
    }
    const int page = kv.block_table[int64_t(seq) * kv.table_stride + in_table];
    if (page < 0 || page >= kv.num_pages) {
        atomicOr(error_flag, kErrBadPage);
        return false;
    }
    tiles = kv.base + int64_t(page) * kv.page_bytes + int64_t(block - in_table * kv.blocks_per_page) * kv.nkvh * kv.tile_bytes;
    return true;
}

} // namespace llaisys::kernels
