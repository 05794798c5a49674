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
// Tokens, list entries and rows of a call: a loop over them looks up to 64 entries, or one step of
// a row loop over the largest grid (65535 CTAs of 160 threads), past the last within 32 bits.
constexpr int32_t kMostEntries = INT32_MAX - (1 << 16);
constexpr int32_t kMostRows = INT32_MAX - (1 << 24);

struct Cache {
    uint8_t *storage;
    int32_t layers;
    int32_t num_blocks;
};

inline Cache cache_of(const void *storage, int32_t layers, int32_t num_blocks) {
    return {static_cast<uint8_t *>(const_cast<void *>(storage)), layers, num_blocks};
}

// The attention of a prompt chunk as rows of the decode attention (arguments checked by the
// caller), and its workspace.
int rows_workspace(int device, int start, int tokens, int64_t *bytes);
int attend_rows(const Cache &cache, int32_t layer, const void *query, bool query_fp32, int64_t query_stride,
                const int32_t *blocks, int32_t start, int32_t tokens, void *out, int64_t out_stride, void *workspace,
                int64_t workspace_bytes, int32_t *error_flag, cudaStream_t stream);

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

// A group's scale as the divisor of its values.
struct Divisor {
    float scale, inverse;

    __device__ __forceinline__ explicit Divisor(uint32_t byte) {
        scale = byte == 0 ? 1.f : scale_value(byte);
        inverse = __frcp_rn(scale);
    }
    // The code of x, plus 8.  x / s is rounded as a division rounds it, since ties must stay ties:
    // from 1 / s, correctly rounded, a quotient within a unit of its last place takes one exact
    // remainder (Markstein's theorem; nothing here is near the ends of FP32's range).
    __device__ __forceinline__ uint32_t code(float x) const {
        const float q = x * inverse;
        const float quotient = fmaf(fmaf(-q, scale, x), inverse, q);
        // The sum's unit is 1: the nearest integer, ties to even, plus 8, in its low bits.
        return __float_as_uint(fminf(fmaxf(quotient, -7.f), 7.f) + (0x1.8p23f + 8.f)) & 15u;
    }
};

__device__ __forceinline__ uint32_t rotate_halves(uint32_t word) {
    return ((word << 2) & 0xfffcfffcu) | ((word >> 14) & 0x00030003u);
}

// Dims 2 l and 2 l + 1 of a token's 64, by the lanes l of a warp, to the word of codes of
// the lane's eight dims (the same in the four lanes that share them) and its group's scale.
__device__ __forceinline__ void encode_pair(float x, float y, int lane, uint32_t &word, uint32_t &scale) {
    uint32_t top = max(__float_as_uint(x) & 0x7fffffffu, __float_as_uint(y) & 0x7fffffffu);
#pragma unroll
    for (int offset = 1; offset < 8; offset <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, offset));
    scale = scale_of(top);
    const Divisor by(scale);
    word = (by.code(x) | by.code(y) << 16) << (4 * (lane & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word = rotate_halves(word);
}

// Dims 8 c .. + 7 of a token, by lane c of its eight, to their word and their group's scale.
__device__ __forceinline__ void encode_chunk(const float (&v)[8], uint32_t &word, uint32_t &scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    scale = scale_of(top);
    const Divisor by(scale);
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= by.code(v[i]) << (4 * (i >> 1) + 16 * (i & 1));
    word = rotate_halves(word);
}

// Byte offsets in a (block, head) of one token's words and scale in group t.
__device__ __forceinline__ int key_words(int t, int token) { return t * (PKV_BLOCK_TOKENS * 8) + token * 8; }
__device__ __forceinline__ int value_word(int chunk, int token) {
    return kValueAt + chunk * (PKV_BLOCK_TOKENS * 4) + token * 4;
}
__device__ __forceinline__ int scale_at(int first, int t, int token) { return first + t * PKV_BLOCK_TOKENS + token; }

// The word of chunk c of a token, and in even chunks its group's scale, into the (block, head) at `head`.
__device__ __forceinline__ void store_key(uint8_t *head, int c, int token, uint32_t word, uint32_t scale) {
    *reinterpret_cast<uint32_t *>(head + key_words(c >> 1, token) + 4 * (c & 1)) = word;
    if ((c & 1) == 0) head[scale_at(kKeyScaleAt, c >> 1, token)] = static_cast<uint8_t>(scale);
}

__device__ __forceinline__ void store_value(uint8_t *head, int c, int token, uint32_t word, uint32_t scale) {
    *reinterpret_cast<uint32_t *>(head + value_word(c, token)) = word;
    if ((c & 1) == 0) head[scale_at(kValueScaleAt, c >> 1, token)] = static_cast<uint8_t>(scale);
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

// What turns a K row: dims 2 l and 2 l + 1 of the norm's weights and of the rotation, by lane.
struct KeyTurn {
    float2 weight, cos, sin;  // sin negative in the lower half of the dims

    __device__ __forceinline__ KeyTurn(const __half *norm, const __half *rope, int position, int lane) {
        constexpr int kHalf = PKV_HEAD_DIM / 2;
        weight = cos = sin = make_float2(0.f, 0.f);
        if (rope == nullptr) return;
        const __half *at = rope + position * kHalf + (2 * lane) % kHalf;
        cos = __half22float2(*reinterpret_cast<const __half2 *>(at));
        sin = __half22float2(*reinterpret_cast<const __half2 *>(at + PKV_CONTEXT_LIMIT * kHalf));
        if (lane < 16) sin = make_float2(-sin.x, -sin.y);
        if (norm != nullptr) weight = __half22float2(*reinterpret_cast<const __half2 *>(norm + 2 * lane));
    }
};

// Dims 2 l and 2 l + 1 of a K row as it is stored, by the lanes l of a warp: with NORM the norm
// of the head (x * rsqrt(mean(x^2) + eps) * weight) first, then the rotation.  The norm is taken
// in FP64: its result is rounded to codes next, and a value beside the border between two must
// not depend on the order of a sum (0.25 us of 8.3 of a decode layer of 7 rows).  Without it FP32 is enough: products of
// FP16 numbers are exact in it, so each rotated value is rounded once.
template <bool NORM>
__device__ __forceinline__ float2 turn_key(__half2 row, const KeyTurn &turn, double eps) {
    const float2 x = __half22float2(row);
    if constexpr (!NORM) {
        const uint32_t far = __shfl_xor_sync(0xffffffffu, pack_half2(row), 16);
        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&far));
        return make_float2(x.x * turn.cos.x + y.x * turn.sin.x, x.y * turn.cos.y + y.y * turn.sin.y);
    }
    const double a = x.x, b = x.y;
    double sum = fma(a, a, b * b);
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    const double inverse = rsqrt(sum * (1.0 / PKV_HEAD_DIM) + eps);
    const double u = a * inverse * static_cast<double>(turn.weight.x), v = b * inverse * static_cast<double>(turn.weight.y);
    const double far_u = __shfl_xor_sync(0xffffffffu, u, 16), far_v = __shfl_xor_sync(0xffffffffu, v, 16);
    return make_float2(static_cast<float>(u * static_cast<double>(turn.cos.x) + far_u * static_cast<double>(turn.sin.x)),
                       static_cast<float>(v * static_cast<double>(turn.cos.y) + far_v * static_cast<double>(turn.sin.y)));
}

}  // namespace pkv::int4
