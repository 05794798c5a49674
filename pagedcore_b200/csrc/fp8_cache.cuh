// Layout of the 8-bit KV cache, and what its sources share on the host.
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
#include <cuda_runtime.h>
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

inline Cache cache_of(const void *key_codes, const void *value_codes, const void *key_scales, const void *value_scales,
                      int32_t layers, int32_t num_blocks) {
    return {static_cast<uint8_t *>(const_cast<void *>(key_codes)), static_cast<uint8_t *>(const_cast<void *>(value_codes)),
            static_cast<float *>(const_cast<void *>(key_scales)), static_cast<float *>(const_cast<void *>(value_scales)),
            layers, num_blocks};
}

// The checks of a cache that every entry point makes.
int check_cache(const void *key_codes, const void *value_codes, const void *key_scales, const void *value_scales,
                int32_t layers, int32_t num_blocks, int32_t layer_begin, int32_t layer_count);

// The new token of every row of a staged batch at `layer`: K rotated and V written, Q
// rotated to query_out + query_low (FP16 numbers that add up to half of the FP32 value).
int launch_decode_append(const Cache &cache, int32_t layer, const void *key, const void *value, int64_t kv_stride,
                         const void *rope_table, const void *query, int64_t query_stride, void *query_out, void *query_low,
                         const int32_t *lengths, const int32_t *prefix, const int32_t *flat, int32_t batch,
                         int32_t total_blocks, int32_t *error_flag, cudaStream_t stream);

}  // namespace pkv::fp8
