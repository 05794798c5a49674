// The 4-bit KV cache: its numbers, its layout, and what its sources share.
//
// A group is 16 consecutive dims of one token and head, stored as 16 codes of 4 bits and
// one scale s of 8 bits; the value of a code c in -7 .. 7 is c * s.
//
// Scale: an unsigned number with 5 exponent and 3 fraction bits, the FP16 number whose bits
// 14 .. 7 its byte is.  It is the one nearest to a seventh of the group's largest magnitude,
// so that the largest over s is at most 7 * 17 / 16 = 7.44 and still rounds to 7: no value
// moves by more than half a step.  Below 2^-14, where the numbers are 2^-17 apart, it is the
// next one up, and past 9216 it stays there (7 * 9216 = 64512 ends inside FP16; the next
// would not): larger values are held at 64512.  Every value is an FP16 number, 7 bits at
// most over 2^-17.  A group with a value that is not finite has the scale 0xff, a NaN.
//
// Codes are uniform because in groups of 16 the largest value is only about twice the root
// mean square: on normal values 7 equal steps leave half the error of the 4-bit float with
// the same scales (5.5e-3 against 1.1e-2 of the variance), and a subtraction decodes them.
//
// Layout: bytes [layers][num_blocks][4 heads][1152], a (block, head) being
//   K codes   512  [4 groups][16 tokens][8 bytes]
//   V codes   512  [8 chunks of 8 dims][16 tokens][4 bytes]
//   K scales   64  [4 groups][16 tokens]
//   V scales   64  [4 groups][16 tokens]
// which is the order in which the lanes of an m16n8k16 MMA want them: lane (g, t) reads K
// of tokens 2 g, 2 g + 1 in group t, 16 bytes, and V of tokens 4 t .. 4 t + 3 in chunk g, 16
// bytes, a warp 512 consecutive bytes each.  A token's own bytes are no other token's, so
// that a write never reads.
//
// Eight codes (dims d .. d + 7 of a token) are a 32-bit word: dim d + 2 i + h is nibble i of its
// 16-bit half h, held as code + 8, and each half is rotated left by two bits.  So rotated,
// nibbles 0 and 1 lie at bits 5 .. 2 and 9 .. 6, and nibbles 2 and 3 do when the bytes of the
// half are swapped: inside the fraction of the FP16 numbers 256 and 16, where a nibble n
// reads as 256 + n or 16 + n.  Two codes take one AND-OR and one multiply-add.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pagedkv.h"
#include "ptx.cuh"

namespace pkv::int4 {

constexpr int kGroup = 16;  // dims per scale
constexpr int kTileBytes = PKV_BLOCK_TOKENS * PKV_HEAD_DIM / 2;  // codes of K or V of one block and head
constexpr int kScaleBytes = PKV_BLOCK_TOKENS * PKV_HEAD_DIM / kGroup;
constexpr int kValueAt = kTileBytes;
constexpr int kKeyScaleAt = 2 * kTileBytes;
constexpr int kValueScaleAt = kKeyScaleAt + kScaleBytes;
constexpr int kHeadBytes = kValueScaleAt + kScaleBytes;
constexpr int kBlockBytes = PKV_KV_HEADS * kHeadBytes;
static_assert(kBlockBytes == PKV_INT4_BLOCK_BYTES, "the header gives the bytes of a block");
constexpr uint32_t kLargestScale = 225;  // 9216
constexpr uint32_t kNanScale = 255;

struct Cache {
    uint8_t *storage;
    int32_t layers;
    int32_t num_blocks;
};

inline Cache cache_of(const void *storage, int32_t layers, int32_t num_blocks) {
    return {static_cast<uint8_t *>(const_cast<void *>(storage)), layers, num_blocks};
}

// The checks of a cache that every entry point makes.
int check_cache(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer_begin, int32_t layer_count);

__device__ __forceinline__ uint8_t *block_at(const Cache &c, int layer, int block) {
    return c.storage + (static_cast<int64_t>(layer) * c.num_blocks + block) * kBlockBytes;
}

// The scale of a group whose magnitudes' largest bit pattern is `top` (NaN is above
// infinity, infinity above every number).
__device__ __forceinline__ uint32_t scale_of(uint32_t top) {
    if (top >= 0x7f800000u) return kNanScale;
    const float seventh = __fdiv_rn(__uint_as_float(top), 7.f);
    if (seventh < 0x1p-14f) return static_cast<uint32_t>(__float2int_ru(seventh * 0x1p17f));
    const uint32_t bits = __float_as_uint(seventh);
    return min((bits + 0x7ffffu + ((bits >> 20) & 1u)) >> 20, kLargestScale + (112u << 3)) - (112u << 3);
}

__device__ __forceinline__ float scale_value(uint32_t scale) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(scale << 7)));
}

// A group's 16 values to its two words of codes and its scale.
__device__ __forceinline__ void encode_group(const float (&v)[16], uint32_t (&words)[2], uint32_t &scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    scale = scale_of(top);
    // x / s rounded as a division rounds it, since ties must stay ties: from 1 / s, correctly
    // rounded, a quotient within a unit of its last place takes one exact remainder (Markstein's
    // theorem; nothing here is near the ends of FP32's range).
    const float s = scale == 0 ? 1.f : scale_value(scale), inverse = __frcp_rn(s);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = v[8 * w + i], q = x * inverse;
            const float quotient = fmaf(fmaf(-q, s, x), inverse, q);
            // The sum's unit is 1: the nearest integer, ties to even, plus 8, in its low bits.
            const uint32_t code = __float_as_uint(fminf(fmaxf(quotient, -7.f), 7.f) + (0x1.8p23f + 8.f));
            word |= (code & 15u) << (4 * (i >> 1) + 16 * (i & 1));
        }
        words[w] = ((word << 2) & 0xfffcfffcu) | ((word >> 14) & 0x00030003u);
    }
}

// Byte offsets in a (block, head) of one token's words and scale in group t.
__device__ __forceinline__ int key_words(int t, int token) { return t * (PKV_BLOCK_TOKENS * 8) + token * 8; }
__device__ __forceinline__ int value_word(int chunk, int token) {
    return kValueAt + chunk * (PKV_BLOCK_TOKENS * 4) + token * 4;
}
__device__ __forceinline__ int scale_at(int first, int t, int token) { return first + t * PKV_BLOCK_TOKENS + token; }

// One group of a token into the (block, head) at `head`, memory of either kind.
__device__ __forceinline__ void store_key(uint8_t *head, int t, int token, const uint32_t (&words)[2], uint32_t scale) {
    *reinterpret_cast<uint2 *>(head + key_words(t, token)) = make_uint2(words[0], words[1]);
    head[scale_at(kKeyScaleAt, t, token)] = static_cast<uint8_t>(scale);
}

__device__ __forceinline__ void store_value(uint8_t *head, int t, int token, const uint32_t (&words)[2], uint32_t scale) {
    *reinterpret_cast<uint32_t *>(head + value_word(2 * t, token)) = words[0];
    *reinterpret_cast<uint32_t *>(head + value_word(2 * t + 1, token)) = words[1];
    head[scale_at(kValueScaleAt, t, token)] = static_cast<uint8_t>(scale);
}

// The FP16 pairs 256 + n (nibbles 0, 2) and 16 + n (nibbles 1, 3) of a word; `swapped` is the word
// with the bytes of each half swapped.
__device__ __forceinline__ __half2 nibble_pair(uint32_t word, uint32_t swapped, int i) {
    const uint32_t from = i < 2 ? word : swapped;
    uint32_t bits;  // (from & mask) | base as one instruction, which the compiler does not make of it
    if (i & 1) asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(bits) : "r"(from), "n"(0x03c003c0), "n"(0x4c004c00));
    else asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(bits) : "r"(from), "n"(0x003c003c), "n"(0x5c005c00));
    return *reinterpret_cast<const __half2 *>(&bits);
}

__device__ __forceinline__ uint32_t swap_bytes(uint32_t word) { return __byte_perm(word, 0, 0x2301); }

// 16 FP16 values at `p` (16-byte aligned) as FP32.
__device__ __forceinline__ void load16(const __half *p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 raw = reinterpret_cast<const uint4 *>(p)[i];
        const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(h[j]);
            v[8 * i + 2 * j] = f.x;
            v[8 * i + 2 * j + 1] = f.y;
        }
    }
}

// Dims 16 t .. + 15 of a K row as it is stored: with `weight` the norm of the head
// (x * rsqrt(mean(x^2) + eps) * weight) first, with `rope` the rotation at `position`.  The
// four lanes of a row call it together; `here` says whether there is a row.  The norm is
// taken in FP64: its result is rounded to codes next, and a value beside the border between
// two must not depend on the order of a sum (60 such operations a lane, which cost nothing
// beside the loads).  Without it FP32 is enough: products of FP16 numbers are exact in it, so
// each rotated value is rounded once.
__device__ __forceinline__ void key_group(const __half *row, int t, bool here, const __half *weight, double eps,
                                          const __half *rope, int position, float (&v)[16]) {
    constexpr int kHalf = PKV_HEAD_DIM / 2;
    float other[16];  // the dims that rotate with these, 32 away
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = other[i] = 0.f;
    if (here) load16(row + kGroup * t, v);
    if (rope == nullptr) return;
    if (here) load16(row + kGroup * (t ^ 2), other);
    float cos[16], sin[16];
    load16(rope + position * kHalf + kGroup * (t & 1), cos);
    load16(rope + (PKV_CONTEXT_LIMIT + position) * kHalf + kGroup * (t & 1), sin);
#pragma unroll
    for (int i = 0; i < 16; ++i) sin[i] = t < 2 ? -sin[i] : sin[i];
    if (weight == nullptr) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = v[i] * cos[i] + other[i] * sin[i];
        return;
    }
    double part[4] = {0, 0, 0, 0};  // four short chains
#pragma unroll
    for (int i = 0; i < 16; ++i) part[i & 3] = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), part[i & 3]);
    double sum = (part[0] + part[1]) + (part[2] + part[3]);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const double inverse = rsqrt(sum * (1.0 / PKV_HEAD_DIM) + eps);
    float own[16], far[16];
    load16(weight + kGroup * t, own);
    load16(weight + kGroup * (t ^ 2), far);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const double x = v[i] * inverse * static_cast<double>(own[i]);
        const double y = other[i] * inverse * static_cast<double>(far[i]);
        v[i] = static_cast<float>(x * static_cast<double>(cos[i]) + y * static_cast<double>(sin[i]));
    }
}

}  // namespace pkv::int4
