// Layout of the 8-bit KV cache, and the RoPE step its kernels share.
//
//   key_codes    [layers][num_blocks][4 heads][16 tokens][64 dims]
//   value_codes  [layers][num_blocks][4 heads][64 dims][16 tokens]
//   key_scales, value_scales  FP32 [layers][num_blocks][4 heads]
//
// A (block, head) tile is 1 KiB and has one scale.  V tiles are transposed:
// the P.V product sums over tokens, and 8-bit codes are turned into MMA
// operands in registers, where the summed index has to be the contiguous one.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "fp8.cuh"
#include "pagedkv.h"

namespace pkv::fp8 {

constexpr int kTileBytes = PKV_BLOCK_TOKENS * PKV_HEAD_DIM;  // 1 KiB: codes of one block and head

struct Cache {
    uint8_t *key_codes;
    uint8_t *value_codes;
    float *key_scales;
    float *value_scales;
    int32_t layers;
    int32_t num_blocks;
};

// Index of a (layer, block, head) tile, in tiles.
__device__ __forceinline__ int64_t tile_index(const Cache &c, int layer, int block, int head) {
    return (static_cast<int64_t>(layer) * c.num_blocks + block) * PKV_KV_HEADS + head;
}

}  // namespace pkv::fp8
