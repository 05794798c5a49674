// Writes to and reads from the 8-bit KV cache (layout: fp8_cache.cuh).
//
// pkv_fp8_append_kv puts new K (optionally rotated) and V rows into their
// slots.  A (block, head) tile has one scale: the tokens that open a block
// (slot 0) set it, later tokens raise it when their magnitudes need more, and
// the codes already in the tile are then rounded again to the larger scale (a
// power of two: only codes near the subnormals change).  Writing the same
// token to the same slot twice leaves the same bytes.
//
// A CTA takes one token of a layer (eight of a long list) with a warp per (K or V,
// head); others, behind them in the grid, rotate the queries.  The warps of a token
// that opens a run (the first token, or one whose slot does not follow the
// previous token's within its block) write the whole run; the tokens of a run
// are those that follow it slot by slot in the block.  K: lane (r, h) holds the
// 32 dims of slot r that rotate together; V: lane l holds dims 2l, 2l + 1 of
// all 16 slots, the two code rows that it stores.  RoPE is computed in FP32
// from the FP16 table and rounded once, to E4M3 (K) or FP16 (Q).  At decode
// the kernel is bound by the latency of its dependent loads (slot, position,
// then row and tile); over a prompt by memory.

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "fp8_cache.cuh"
#include "pdl.h"
#include "prefill_attention.h"
#include "ptx.cuh"
#include "status.h"

namespace {

constexpr int kDim = PKV_HEAD_DIM;
constexpr int kHalf = kDim / 2;
constexpr int kHeads = PKV_KV_HEADS;
constexpr int kSlots = PKV_BLOCK_TOKENS;
constexpr int kThreads = 2 * kHeads * 32;

struct AppendArgs {
    pkv::fp8::Cache cache;
    int32_t layer_begin;
    const __half *key;
    const __half *value;
    int64_t layer_stride;
    int64_t token_stride;
    const int32_t *slots;
    const int32_t *positions;  // with rope
    int32_t tokens;
    const __half *rope;  // FP16 cos [2048][32], sin [2048][32], or null
    const __half *query_in;
    __half *query_out;
    __half *query_low;   // nullable, laid out as query_out: then both hold halves of the values
                         // (two FP16 components can rotate past FP16's range), and this what FP16 left of each
    float *query_out32;  // in place of query_out: the rotated queries in FP32
    int64_t q_layer_stride;
    int64_t q_token_stride;
    int64_t q_out_layer_stride;
    int64_t q_out_token_stride;
    int32_t *error_flag;
    // A staged decode batch: token b is row b's new one, at position lengths[b] - 1 in
    // the last of its blocks flat[prefix[b] .. prefix[b + 1]); slots and positions unused.
    const int32_t *lengths;
    const int32_t *prefix;
    const int32_t *flat;
    int32_t total_blocks;
    int32_t tile_ctas;  // CTAs that write K and V; those that rotate queries come after them in the grid
    int32_t span;       // tokens per CTA of the former
};

constexpr int kQuerySpan = 4;  // tokens per CTA that rotates queries

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, offset));
    return v;
}

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

// RoPE of dims d .. d+15 (lo) and d+32 .. d+47 (hi) at `position`.
__device__ __forceinline__ void rotate16(const __half *rope, int position, int d, float (&lo)[16], float (&hi)[16]) {
    float c[16], s[16];
    load16(rope + position * kHalf + d, c);
    load16(rope + (PKV_CONTEXT_LIMIT + position) * kHalf + d, s);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float a = lo[i], b = hi[i];
        lo[i] = a * c[i] - b * s[i];
        hi[i] = b * c[i] + a * s[i];
    }
}

__device__ __forceinline__ int checked_position(const AppendArgs &a, int token) {
    const int position = a.lengths != nullptr ? a.lengths[token] - 1 : a.positions[token];
    if (position >= 0 && position < PKV_CONTEXT_LIMIT) return position;
    atomicOr(a.error_flag, PKV_DEVICE_BAD_POSITION);
    return 0;
}

// The token's slot, or -1.
__device__ __forceinline__ int slot_of(const AppendArgs &a, int token) {
    int slot;
    if (a.lengths != nullptr) {
        const int last = a.prefix[token + 1], length = a.lengths[token];
        const int block = last >= 1 && last <= a.total_blocks ? a.flat[last - 1] : -1;
        slot = block >= 0 && block < a.cache.num_blocks && length >= 1 && length <= PKV_CONTEXT_LIMIT
                   ? block * kSlots + (length - 1) % kSlots
                   : -1;
    } else {
        slot = a.slots[token];
    }
    return slot < static_cast<int64_t>(a.cache.num_blocks) * kSlots ? slot : -1;
}

// 16 values to 16 codes.
__device__ __forceinline__ uint4 encode16(const float (&v)[16], float inverse, bool largest) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = pkv::fp8::scaled(v[4 * i + j], inverse, largest);
        w[i] = pkv::fp8::encode2(s[0], s[1]) | (pkv::fp8::encode2(s[2], s[3]) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 rescale16(const uint4 &c, float factor) {
    return make_uint4(pkv::fp8::rescale4(c.x, factor), pkv::fp8::rescale4(c.y, factor),
                      pkv::fp8::rescale4(c.z, factor), pkv::fp8::rescale4(c.w, factor));
}

// Exponent for a tile whose new values reach `amax`: the held one is kept or
// raised, unless the tile's first slot is being written.
__device__ __forceinline__ int tile_exponent(float amax, int first_slot, float held, int &held_exponent) {
    const int needed = pkv::fp8::scale_exponent(amax);
    held_exponent = first_slot > 0 ? pkv::fp8::stored_exponent(held) : needed;
    return max(needed, held_exponent);
}

__device__ void write_key(const AppendArgs &a, int layer, int head, int token, int run, int block, int first,
                          int lane) {
    const int64_t tile = pkv::fp8::tile_index(a.cache, layer + a.layer_begin, block, head);
    uint8_t *codes = a.cache.key_codes + tile * pkv::fp8::kTileBytes;
    const float held_scale = first > 0 ? a.cache.key_scales[tile] : 0.f;
    const int r = lane >> 1, d = 16 * (lane & 1);
    const bool fresh = r >= first && r < first + run;
    float lo[16], hi[16];
    float amax = 0.f;
    if (fresh) {
        const int t = token + r - first;
        const __half *src = a.key + layer * a.layer_stride + t * a.token_stride + head * kDim + d;
        load16(src, lo);
        load16(src + kHalf, hi);
        if (a.rope != nullptr) rotate16(a.rope, checked_position(a, t), d, lo, hi);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = pkv::fp8::max_finite(pkv::fp8::max_finite(amax, lo[i]), hi[i]);
    }
    amax = warp_max(amax);
    int held;
    const int e = tile_exponent(amax, first, held_scale, held);
    uint4 *row = reinterpret_cast<uint4 *>(codes + r * kDim + d);
    if (fresh) {
        const float inverse = pkv::fp8::exp2_int(-e);
        const bool largest = e == pkv::fp8::kMaxExponent;
        row[0] = encode16(lo, inverse, largest);
        row[kHalf / 16] = encode16(hi, inverse, largest);
    } else if (r < first && e > held) {
        const float factor = pkv::fp8::exp2_int(held - e);
        row[0] = rescale16(row[0], factor);
        row[kHalf / 16] = rescale16(row[kHalf / 16], factor);
    }
    __syncwarp();  // every lane has read the held scale
    if (lane == 0) a.cache.key_scales[tile] = pkv::fp8::exp2_int(e);
}

__device__ void write_value(const AppendArgs &a, int layer, int head, int token, int run, int block, int first,
                            int lane) {
    const int64_t tile = pkv::fp8::tile_index(a.cache, layer + a.layer_begin, block, head);
    uint4 *rows = reinterpret_cast<uint4 *>(a.cache.value_codes + tile * pkv::fp8::kTileBytes) + 2 * lane;
    const float held_scale = first > 0 ? a.cache.value_scales[tile] : 0.f;
    const uint4 stored[2] = {rows[0], rows[1]};
    const __half *src = a.value + layer * a.layer_stride + token * a.token_stride + head * kDim + 2 * lane;
    float v[2][kSlots];  // of dims 2 lane, 2 lane + 1 by slot
    float amax = 0.f;
#pragma unroll
    for (int r = 0; r < kSlots; ++r) {
        float2 f = make_float2(0.f, 0.f);
        if (r >= first && r < first + run) {
            f = __half22float2(*reinterpret_cast<const __half2 *>(src + (r - first) * a.token_stride));
            amax = pkv::fp8::max_finite(pkv::fp8::max_finite(amax, f.x), f.y);
        }
        v[0][r] = f.x;
        v[1][r] = f.y;
    }
    amax = warp_max(amax);
    int held;
    const int e = tile_exponent(amax, first, held_scale, held);
    const float inverse = pkv::fp8::exp2_int(-e);
    const bool largest = e == pkv::fp8::kMaxExponent;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 fresh = encode16(v[i], inverse, largest);
        uint4 codes = stored[i];
        const uint32_t *f = reinterpret_cast<const uint32_t *>(&fresh);
        uint32_t *c = reinterpret_cast<uint32_t *>(&codes);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t again = c[q];
            if (e > held) again = pkv::fp8::rescale4(again, pkv::fp8::exp2_int(held - e));
            uint32_t word = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 4 * q + j;
                const uint32_t from = r < first ? again : r < first + run ? f[q] : c[q];
                word |= from & (0xffu << (8 * j));
            }
            c[q] = word;
        }
        rows[i] = codes;
    }
    __syncwarp();
    if (lane == 0) a.cache.value_scales[tile] = pkv::fp8::exp2_int(e);
}

// RoPE of kQuerySpan tokens' queries, four heads a warp: eight lanes a head, eight
// dims a lane; the partner's dims (32 away) come from the lane four further.
__device__ void rotate_queries(const AppendArgs &a, int layer, int begin, int warp, int lane) {
    const int chunk = lane & 7, at = (4 * warp + (lane >> 3)) * kDim + 8 * chunk;
    const float sign = chunk < 4 ? -1.f : 1.f;
    uint4 own[kQuerySpan], cos[kQuerySpan], sin[kQuerySpan];
    bool here[kQuerySpan];
#pragma unroll
    for (int j = 0; j < kQuerySpan; ++j) {
        const int token = begin + j;
        here[j] = token < a.tokens && (a.lengths == nullptr || a.prefix[token + 1] > a.prefix[token]);
        own[j] = cos[j] = sin[j] = make_uint4(0, 0, 0, 0);
        if (here[j]) {
            own[j] = *reinterpret_cast<const uint4 *>(a.query_in + layer * a.q_layer_stride + token * a.q_token_stride + at);
            const __half *factors = a.rope + checked_position(a, token) * kHalf + 8 * (chunk & 3);
            cos[j] = *reinterpret_cast<const uint4 *>(factors);
            sin[j] = *reinterpret_cast<const uint4 *>(factors + PKV_CONTEXT_LIMIT * kHalf);
        }
    }
#pragma unroll
    for (int j = 0; j < kQuerySpan; ++j) {
        const uint32_t x[4] = {own[j].x, own[j].y, own[j].z, own[j].w}, c[4] = {cos[j].x, cos[j].y, cos[j].z, cos[j].w},
                       s[4] = {sin[j].x, sin[j].y, sin[j].z, sin[j].w};
        float2 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t p = __shfl_xor_sync(0xffffffffu, x[i], 4);
            const float2 xf = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
            const float2 pf = __half22float2(*reinterpret_cast<const __half2 *>(&p));
            const float2 cf = __half22float2(*reinterpret_cast<const __half2 *>(&c[i]));
            const float2 sf = __half22float2(*reinterpret_cast<const __half2 *>(&s[i]));
            y[i] = make_float2(xf.x * cf.x + sign * pf.x * sf.x, xf.y * cf.y + sign * pf.y * sf.y);
        }
        if (!here[j]) continue;
        const int64_t to = layer * a.q_out_layer_stride + (begin + j) * a.q_out_token_stride + at;
        if (a.query_out32 != nullptr) {
            float4 *dst = reinterpret_cast<float4 *>(a.query_out32 + to);
            dst[0] = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
            dst[1] = make_float4(y[2].x, y[2].y, y[3].x, y[3].y);
            continue;
        }
        uint32_t r[4], low[4];
        const float part = a.query_low != nullptr ? 0.5f : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i].x *= part, y[i].y *= part;
            const __half2 h = __floats2half2_rn(y[i].x, y[i].y);
            const float2 f = __half22float2(h);
            r[i] = pkv::pack_half2(h);
            low[i] = pkv::pack_half2(__floats2half2_rn(y[i].x - f.x, y[i].y - f.y));
        }
        *reinterpret_cast<uint4 *>(a.query_out + to) = make_uint4(r[0], r[1], r[2], r[3]);
        if (a.query_low != nullptr) {
            *reinterpret_cast<uint4 *>(a.query_low + to) = make_uint4(low[0], low[1], low[2], low[3]);
        }
    }
}

// The grid for `tokens`: eight tokens a CTA (of a prompt every sixteenth opens a run) from 512
// tokens on, where a single layer still gives 64 CTAs or more; several layers have a grid row each.
dim3 append_grid(AppendArgs &a, int layers) {
    a.span = a.lengths == nullptr && a.tokens >= 512 ? 8 : 1;
    a.tile_ctas = (a.tokens + a.span - 1) / a.span;
    return dim3(a.tile_ctas + (a.query_in != nullptr ? (a.tokens + kQuerySpan - 1) / kQuerySpan : 0), layers);
}

// Two CTAs an SM: with the 80 registers that three leave, the write of a run spills
// (2047 tokens with queries 10.2 us, 9.4 so; 8.6 and 7.0 without queries).
__global__ void __launch_bounds__(kThreads, 2) fp8_append_kernel(const __grid_constant__ AppendArgs a) {
    // In this order: the decode attention behind it reads what is older than this
    // kernel (the tables, the cache but for the blocks written here) before its own wait.
    pkv::pdl_wait();
    pkv::pdl_launch_dependents();
    const int layer = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (static_cast<int>(blockIdx.x) >= a.tile_ctas) {
        rotate_queries(a, layer, (static_cast<int>(blockIdx.x) - a.tile_ctas) * kQuerySpan, warp, lane);
        return;
    }
    const int begin = static_cast<int>(blockIdx.x) * a.span;
    // Slots of the tokens from begin - 1 on: a span's runs end 15 tokens past it.
    const int near = begin - 1 + lane;
    int slot_at = -1;
    if (near >= 0 && near < a.tokens) slot_at = slot_of(a, near);
    for (int j = 0; j < a.span && begin + j < a.tokens; ++j) {
        const int token = begin + j;
        if (a.lengths != nullptr && a.prefix[token + 1] <= a.prefix[token]) continue;  // a row without blocks
        const int slot = __shfl_sync(0xffffffffu, slot_at, j + 1);
        if (slot < 0) {
            if (threadIdx.x == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
            continue;
        }
        const int first = slot % kSlots;
        int run = 1;
        if (a.lengths == nullptr) {
            const int previous = __shfl_sync(0xffffffffu, slot_at, j);
            if (first != 0 && token > 0 && previous == slot - 1) continue;  // written with its run's first token
            const int ahead = lane - (j + 1);  // of this token
            const bool follows = ahead >= 0 && ahead < kSlots - first && near < a.tokens && slot_at == slot + ahead;
            run = __ffs(~(__ballot_sync(0xffffffffu, follows) >> (j + 1))) - 1;
        }
        if (warp < kHeads) {
            write_key(a, layer, warp, token, run, slot / kSlots, first, lane);
        } else {
            write_value(a, layer, warp - kHeads, token, run, slot / kSlots, first, lane);
        }
    }
}

// K and V of `blocks` as FP16, each [i][slot][head][dim].  One CTA per block: K code rows go straight across; V tiles turn around in shared memory.
// index_out (nullable) receives 0 .. count - 1, the block table of the outputs as a pool.
constexpr int kReadThreads = 256;
constexpr int64_t kBlockValues = kSlots * kHeads * kDim;

__global__ void __launch_bounds__(kReadThreads)
    fp8_read_kernel(const pkv::fp8::Cache cache, int layer, const int32_t *blocks, __half *key_out, __half *value_out,
                    int32_t *index_out, int32_t *error_flag) {
    __shared__ __align__(16) __half turned[kHeads][kSlots][kDim + 8];
    pkv::pdl_launch_dependents();
    pkv::pdl_wait();
    const int block = blocks[blockIdx.x];
    const bool bad = block < 0 || block >= cache.num_blocks;
    if (bad && threadIdx.x == 0) atomicOr(error_flag, PKV_DEVICE_BAD_BLOCK);
    if (index_out != nullptr && threadIdx.x == 0) index_out[blockIdx.x] = blockIdx.x;
    const int head = threadIdx.x >> 6;
    const int part = threadIdx.x & 63;  // 16 codes of the head's tile
    const int64_t tile = bad ? 0 : pkv::fp8::tile_index(cache, layer, block, head);
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    float ks = 0.f, vs = 0.f;
    if (!bad) {
        k = reinterpret_cast<const uint4 *>(cache.key_codes + tile * pkv::fp8::kTileBytes)[part];
        v = reinterpret_cast<const uint4 *>(cache.value_codes + tile * pkv::fp8::kTileBytes)[part];
        ks = cache.key_scales[tile];
        vs = cache.value_scales[tile];
    }
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kBlockValues;
    const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, vw[4] = {v.x, v.y, v.z, v.w};
    __align__(16) __half2 row[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = pkv::fp8::decode2f(kw[i >> 1] >> (16 * (i & 1)));
        row[i] = __floats2half2_rn(f.x * ks, f.y * ks);
        const float2 g = pkv::fp8::decode2f(vw[i >> 1] >> (16 * (i & 1)));
        turned[head][2 * i][part] = __float2half_rn(g.x * vs);  // part is the dim
        turned[head][2 * i + 1][part] = __float2half_rn(g.y * vs);
    }
    uint4 *kd = reinterpret_cast<uint4 *>(key_out + at + ((part >> 2) * kHeads + head) * kDim + (part & 3) * 16);
    kd[0] = reinterpret_cast<const uint4 *>(row)[0];
    kd[1] = reinterpret_cast<const uint4 *>(row)[1];
    __syncthreads();
    for (int i = threadIdx.x; i < kSlots * kHeads * kDim / 8; i += kReadThreads) {
        const int h = (i >> 3) & 3, slot = i >> 5, chunk = i & 7;
        reinterpret_cast<uint4 *>(value_out + at)[i] =
            *reinterpret_cast<const uint4 *>(&turned[h][slot][8 * chunk]);
    }
}

// The open blocks of a step (those of `slots` that are not a block's first), all layers:
// codes and scales to `saved` before the step, or back from it.  One CTA per (slot, layer),
// 16 bytes of K and of V a thread.  256 slots of 22 layers are 46 MB each way.
constexpr int kSavedBytes = 2 * kHeads * pkv::fp8::kTileBytes + 2 * kHeads * 4;  // K codes, V codes, K and V scales

template <bool RESTORE>
__global__ void __launch_bounds__(kReadThreads) fp8_save_kernel(const pkv::fp8::Cache cache, const int32_t *slots,
                                                                uint8_t *saved) {
    pkv::pdl_wait();
    pkv::pdl_launch_dependents();
    const int slot = slots[blockIdx.x];
    if (slot < 0 || slot % kSlots == 0 || slot / kSlots >= cache.num_blocks) return;
    const int64_t tile = pkv::fp8::tile_index(cache, blockIdx.y, slot / kSlots, 0);
    uint4 *const held = reinterpret_cast<uint4 *>(saved + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kSavedBytes);
    const auto copy = [&](void *block, int at, int i) {
        uint4 *const stored = static_cast<uint4 *>(block);
        if (RESTORE) stored[i] = held[at + i];
        else held[at + i] = stored[i];
    };
    constexpr int kCodes = kHeads * pkv::fp8::kTileBytes / 16;  // of K or V
    static_assert(kCodes == kReadThreads, "a thread takes 16 bytes of each");
    copy(cache.key_codes + tile * pkv::fp8::kTileBytes, 0, threadIdx.x);
    copy(cache.value_codes + tile * pkv::fp8::kTileBytes, kCodes, threadIdx.x);
    if (threadIdx.x < 2) copy((threadIdx.x ? cache.value_scales : cache.key_scales) + tile, 2 * kCodes + threadIdx.x, 0);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

namespace pkv::fp8 {

int check_cache(const void *key_codes, const void *value_codes, const void *key_scales, const void *value_scales,
                int32_t layers, int32_t num_blocks, int32_t layer_begin, int32_t layer_count) {
    if (key_codes == nullptr || value_codes == nullptr || key_scales == nullptr || value_scales == nullptr) {
        return fail(PKV_VALUE_ERROR, "fp8 cache: codes and scales are required");
    }
    if (!aligned16(key_codes) || !aligned16(value_codes) || !aligned16(key_scales) || !aligned16(value_scales)) {
        return fail(PKV_VALUE_ERROR, "fp8 cache: codes and scales must be 16-byte aligned");
    }
    if (layers < 1 || num_blocks < 1 || num_blocks > INT32_MAX / PKV_BLOCK_TOKENS) {
        return fail(PKV_VALUE_ERROR, "fp8 cache: layer or block count out of range");
    }
    if (layer_begin < 0 || layer_count < 1 || layer_count > layers - layer_begin) {
        return fail(PKV_VALUE_ERROR, "fp8 cache: layers out of range");
    }
    return PKV_OK;
}

int launch_decode_append(const Cache &cache, int32_t layer, const void *key, const void *value, int64_t kv_stride,
                         const void *rope_table, const void *query, int64_t query_stride, void *query_out, void *query_low,
                         const int32_t *lengths, const int32_t *prefix, const int32_t *flat, int32_t batch,
                         int32_t total_blocks, int32_t *error_flag, cudaStream_t stream) {
    if (!aligned16(key) || !aligned16(value) || kv_stride % 8 || !aligned16(rope_table)) {
        return fail(PKV_VALUE_ERROR, "fp8 decode: new K/V rows must be 16-byte aligned with strides in multiples of 8");
    }
    AppendArgs a = {};
    a.cache = cache;
    a.layer_begin = layer;
    a.key = static_cast<const __half *>(key);
    a.value = static_cast<const __half *>(value);
    a.token_stride = kv_stride;
    a.tokens = batch;
    a.rope = static_cast<const __half *>(rope_table);
    a.query_in = static_cast<const __half *>(query);
    a.query_out = static_cast<__half *>(query_out);
    a.query_low = static_cast<__half *>(query_low);
    a.q_token_stride = query_stride;
    a.q_out_token_stride = PKV_QUERY_HEADS * PKV_HEAD_DIM;
    a.error_flag = error_flag;
    a.lengths = lengths;
    a.prefix = prefix;
    a.flat = flat;
    a.total_blocks = total_blocks;
    const cudaError_t e = launch_pdl(fp8_append_kernel, append_grid(a, 1), dim3(kThreads), stream, a);
    if (e != cudaSuccess) return fail(PKV_CUDA_ERROR, std::string("fp8 append launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

}  // namespace pkv::fp8

extern "C" int pkv_fp8_append_kv(void *key_codes, void *value_codes, void *key_scales, void *value_scales,
                                 int32_t layers, int32_t num_blocks, int32_t layer_begin, int32_t layer_count,
                                 const void *key, const void *value, int64_t src_layer_stride, int64_t src_token_stride,
                                 const int32_t *slots, const int32_t *positions, int32_t tokens, const void *rope_table,
                                 const void *query_in, int64_t q_layer_stride, int64_t q_token_stride, void *query_out,
                                 int32_t query_out_fp32, int64_t q_out_layer_stride, int64_t q_out_token_stride,
                                 int32_t *error_flag, void *stream) {
    pkv::clear_error();
    int rc = pkv::fp8::check_cache(key_codes, value_codes, key_scales, value_scales, layers, num_blocks, layer_begin,
                                   layer_count);
    if (rc) return rc;
    if (key == nullptr || value == nullptr || slots == nullptr || error_flag == nullptr || tokens < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 append: key, value, slots and error_flag are required");
    }
    if ((rope_table != nullptr) != (positions != nullptr) || (query_in != nullptr) != (query_out != nullptr) ||
        (query_in != nullptr && rope_table == nullptr)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 append: rope_table goes with positions, query with both and an output");
    }
    if (!aligned16(key) || !aligned16(value) || src_layer_stride % 8 || src_token_stride % 8 ||
        (rope_table && !aligned16(rope_table)) ||
        (query_in && (!aligned16(query_in) || !aligned16(query_out) || q_layer_stride % 8 || q_token_stride % 8 ||
                      q_out_layer_stride % 8 || q_out_token_stride % 8))) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 append: rows must be 16-byte aligned with strides in multiples of 8");
    }
    if (layer_count > 65535) return pkv::fail(PKV_VALUE_ERROR, "fp8 append: layers out of range");
    if (tokens == 0) return PKV_OK;
    AppendArgs a = {};
    a.cache = pkv::fp8::cache_of(key_codes, value_codes, key_scales, value_scales, layers, num_blocks);
    a.layer_begin = layer_begin;
    a.key = static_cast<const __half *>(key);
    a.value = static_cast<const __half *>(value);
    a.layer_stride = src_layer_stride;
    a.token_stride = src_token_stride;
    a.slots = slots;
    a.positions = positions;
    a.tokens = tokens;
    a.rope = static_cast<const __half *>(rope_table);
    a.query_in = static_cast<const __half *>(query_in);
    a.query_out = query_out_fp32 ? nullptr : static_cast<__half *>(query_out);
    a.query_out32 = query_out_fp32 ? static_cast<float *>(query_out) : nullptr;
    a.query_low = nullptr;
    a.q_layer_stride = q_layer_stride;
    a.q_token_stride = q_token_stride;
    a.q_out_layer_stride = q_out_layer_stride;
    a.q_out_token_stride = q_out_token_stride;
    a.error_flag = error_flag;
    a.lengths = nullptr;
    a.prefix = nullptr;
    a.flat = nullptr;
    a.total_blocks = 0;
    const cudaError_t e = pkv::launch_pdl(fp8_append_kernel, append_grid(a, layer_count), dim3(kThreads),
                                          static_cast<cudaStream_t>(stream), a);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 append launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

namespace {

int read_blocks(const void *key_codes, const void *value_codes, const void *key_scales, const void *value_scales,
                int32_t layers, int32_t num_blocks, int32_t layer, const int32_t *blocks, int32_t count, void *key_out,
                void *value_out, int32_t *index_out, int32_t *error_flag, void *stream) {
    const int rc = pkv::fp8::check_cache(key_codes, value_codes, key_scales, value_scales, layers, num_blocks, layer, 1);
    if (rc) return rc;
    if (blocks == nullptr || key_out == nullptr || value_out == nullptr || error_flag == nullptr || count < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 read: blocks, outputs and error_flag are required");
    }
    if (!aligned16(key_out) || !aligned16(value_out)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 read: the outputs must be 16-byte aligned");
    }
    if (count == 0) return PKV_OK;
    const cudaError_t e = pkv::launch_pdl(
        fp8_read_kernel, dim3(count), dim3(kReadThreads), static_cast<cudaStream_t>(stream),
        pkv::fp8::cache_of(key_codes, value_codes, key_scales, value_scales, layers, num_blocks), layer, blocks,
        static_cast<__half *>(key_out), static_cast<__half *>(value_out), index_out, error_flag);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 read launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

}  // namespace

extern "C" int pkv_fp8_read_blocks(const void *key_codes, const void *value_codes, const void *key_scales,
                                   const void *value_scales, int32_t layers, int32_t num_blocks, int32_t layer,
                                   const int32_t *blocks, int32_t count, void *key_out, void *value_out,
                                   int32_t *error_flag, void *stream) {
    pkv::clear_error();
    return read_blocks(key_codes, value_codes, key_scales, value_scales, layers, num_blocks, layer, blocks, count,
                       key_out, value_out, nullptr, error_flag, stream);
}

extern "C" int pkv_fp8_save_blocks(void *key_codes, void *value_codes, void *key_scales, void *value_scales,
                                   int32_t layers, int32_t num_blocks, const int32_t *slots, int32_t count, void *saved,
                                   int64_t saved_bytes, int32_t restore, void *stream) {
    pkv::clear_error();
    const int rc = pkv::fp8::check_cache(key_codes, value_codes, key_scales, value_scales, layers, num_blocks, 0, layers);
    if (rc) return rc;
    if (slots == nullptr || saved == nullptr || count < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 save: slots and a buffer are required");
    }
    if (layers > 65535) return pkv::fail(PKV_VALUE_ERROR, "fp8 save: layers out of range");
    if (!aligned16(saved) || saved_bytes / kSavedBytes / layers < count) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 save: the buffer must be 16-byte aligned, 8224 bytes for each layer and slot");
    }
    if (count == 0) return PKV_OK;
    const cudaError_t e = pkv::launch_pdl(restore ? fp8_save_kernel<true> : fp8_save_kernel<false>, dim3(count, layers),
                                          dim3(kReadThreads), static_cast<cudaStream_t>(stream),
                                          pkv::fp8::cache_of(key_codes, value_codes, key_scales, value_scales, layers, num_blocks),
                                          slots, static_cast<uint8_t *>(saved));
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 save launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

// The request's blocks become an FP16 pool of one layer in the workspace (the values are
// FP16 numbers: nothing is rounded), which the tensor-core prompt kernel attends to.  That
// kernel reads every block once for each 16 queries, so the conversion is a small part: 2 of
// 53 us at 2047 tokens.  (The prompt kernel's producers reading codes and converting them, every
// block as often as there are 16 queries behind it, took 16 to 27 us more for 2047 tokens, 5 for
// 75 behind 601.)
extern "C" int pkv_fp8_prefill_attention(const void *key_codes, const void *value_codes, const void *key_scales,
                                         const void *value_scales, int32_t layers, int32_t num_blocks, int32_t layer,
                                         const void *query, int32_t query_fp32, int64_t query_stride,
                                         const int32_t *blocks, int32_t start, int32_t tokens, void *out,
                                         int64_t out_stride, void *workspace, int64_t workspace_bytes,
                                         int32_t *error_flag, void *stream) {
    pkv::clear_error();
    if (query == nullptr || blocks == nullptr || out == nullptr || error_flag == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: null pointer argument");
    }
    if (tokens < 1 || start < 0 || static_cast<int64_t>(start) + tokens > PKV_CONTEXT_LIMIT) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: the chunk must hold 1 or more tokens at positions below 2048");
    }
    constexpr int64_t kRow = PKV_QUERY_HEADS * PKV_HEAD_DIM;
    if (!aligned16(query) || !aligned16(out) || query_stride % 8 || out_stride % 8 || query_stride < kRow ||
        out_stride < kRow) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: rows must be 16-byte aligned, 2048 or more values apart in multiples of 8");
    }
    const int count = (start + tokens + kSlots - 1) / kSlots;
    const int64_t pool_bytes = static_cast<int64_t>(count) * 2 * kBlockValues * 2;
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < pool_bytes + 4 * count) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: the workspace needs 16388 bytes per block of 16 tokens");
    }
    int32_t *const table = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(workspace) + pool_bytes);
    const int rc = read_blocks(key_codes, value_codes, key_scales, value_scales, layers, num_blocks, layer, blocks, count,
                               workspace, static_cast<__half *>(workspace) + count * kBlockValues, table, error_flag,
                               stream);
    if (rc) return rc;
    return pkv::launch_prefill_attention_tc(workspace, count, 0, query, query_fp32 != 0, true, query_stride, table, start,
                                            tokens, out, out_stride, error_flag, static_cast<cudaStream_t>(stream));
}
