// Writes to and reads from the 4-bit KV cache (numbers and layout: int4.cuh).
//
// pkv_int4_append_kv puts new K (with a norm of each head and the rotation, where asked for)
// and V rows into their slots.  A warp takes K or V of one head of four tokens, a lane eight
// dims, which are a word of codes; consecutive tokens of a block fill whole sectors.  Tokens
// are independent of one another.  CTAs behind those rotate the queries.

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "int4.cuh"
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
constexpr int kSpan = 4;       // tokens per CTA that writes K and V
constexpr int kQuerySpan = 2;  // and per CTA that rotates queries

struct AppendArgs {
    pkv::int4::Cache cache;
    int32_t layer_begin;
    const __half *key;
    const __half *value;
    int64_t layer_stride;
    int64_t token_stride;
    const int32_t *slots;
    const int32_t *positions;  // with rope
    int32_t tokens;
    const __half *rope;        // FP16 cos [2048][32], sin [2048][32], or null
    const __half *query_norm;  // FP16 [layers][64], or null
    const __half *key_norm;
    double eps;
    const __half *query_in;
    void *query_out;
    int32_t query_out_fp32;
    int64_t q_layer_stride;
    int64_t q_token_stride;
    int64_t q_out_layer_stride;
    int64_t q_out_token_stride;
    int32_t *error_flag;
    int32_t tile_ctas;  // CTAs that write K and V; those that rotate queries come after them in the grid
};

__device__ __forceinline__ int checked_position(const AppendArgs &a, int token) {
    const int position = a.positions[token];
    if (position >= 0 && position < PKV_CONTEXT_LIMIT) return position;
    atomicOr(a.error_flag, PKV_DEVICE_BAD_POSITION);
    return 0;
}

__device__ __forceinline__ float4 four(const uint2 &raw) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x));
    const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
    return make_float4(x.x, x.y, y.x, y.y);
}

// Norm and RoPE of kQuerySpan tokens' queries: sixteen lanes a head, four dims a lane, so that
// each store of FP32 fills whole sectors; the partner's dims (32 away) come from the lane eight
// further.  A warp has two pairs of heads of each token in flight.
__device__ void rotate_queries(const AppendArgs &a, int layer, int begin, int warp, int lane) {
    constexpr int kPairs = kQuerySpan * 2;  // (token, pair of heads) of a warp
    const int c = lane & 15;
    const float sign = c < 8 ? -1.f : 1.f;
    float4 weight = make_float4(1.f, 1.f, 1.f, 1.f);
    if (a.query_norm != nullptr) {
        weight = four(*reinterpret_cast<const uint2 *>(a.query_norm + static_cast<int64_t>(a.layer_begin + layer) * kDim + 4 * c));
    }
    uint2 own[kPairs], cos[kPairs], sin[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        const int token = min(begin + j / 2, a.tokens - 1), head = 4 * warp + 2 * (j & 1) + (lane >> 4);
        own[j] = *reinterpret_cast<const uint2 *>(a.query_in + layer * a.q_layer_stride + token * a.q_token_stride + head * kDim + 4 * c);
        const __half *factors = a.rope + checked_position(a, token) * kHalf + 4 * (c & 7);
        cos[j] = *reinterpret_cast<const uint2 *>(factors);
        sin[j] = *reinterpret_cast<const uint2 *>(factors + PKV_CONTEXT_LIMIT * kHalf);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        float4 x = four(own[j]);
        if (a.query_norm != nullptr) {
            float sum = fmaf(x.x, x.x, x.y * x.y) + fmaf(x.z, x.z, x.w * x.w);
#pragma unroll
            for (int offset = 1; offset < 16; offset <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
            const float inverse = rsqrtf(sum * (1.f / kDim) + static_cast<float>(a.eps));
            x.x *= inverse * weight.x, x.y *= inverse * weight.y, x.z *= inverse * weight.z, x.w *= inverse * weight.w;
        }
        const float4 p = make_float4(__shfl_xor_sync(0xffffffffu, x.x, 8), __shfl_xor_sync(0xffffffffu, x.y, 8),
                                     __shfl_xor_sync(0xffffffffu, x.z, 8), __shfl_xor_sync(0xffffffffu, x.w, 8));
        const float4 k = four(cos[j]), s = four(sin[j]);
        const float4 y = make_float4(x.x * k.x + sign * p.x * s.x, x.y * k.y + sign * p.y * s.y,
                                     x.z * k.z + sign * p.z * s.z, x.w * k.w + sign * p.w * s.w);
        const int token = begin + j / 2, head = 4 * warp + 2 * (j & 1) + (lane >> 4);
        if (token >= a.tokens) continue;
        const int64_t to = layer * a.q_out_layer_stride + token * a.q_out_token_stride + head * kDim + 4 * c;
        if (a.query_out_fp32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(a.query_out) + to) = y;
        } else {
            const uint32_t low = pkv::pack_half2(__floats2half2_rn(y.x, y.y)), high = pkv::pack_half2(__floats2half2_rn(y.z, y.w));
            *reinterpret_cast<uint2 *>(static_cast<__half *>(a.query_out) + to) = make_uint2(low, high);
        }
    }
}

// Eight FP16 values as FP32.
__device__ __forceinline__ void halves(const uint4 &raw, float (&v)[8]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}

// turn_key of int4.cuh by the eight lanes c of a row: dims 8 c .. + 7, `raw` in FP16, to v.
__device__ __forceinline__ void turn_chunk(const AppendArgs &a, int layer, int position, int c, const uint4 &raw, float (&v)[8]) {
    const __half *factors = a.rope + position * kHalf + 8 * (c & 3);
    float cos[8], sin[8], far[8];
    halves(*reinterpret_cast<const uint4 *>(factors), cos);
    halves(*reinterpret_cast<const uint4 *>(factors + PKV_CONTEXT_LIMIT * kHalf), sin);
    uint4 other;  // the dims that rotate with these, 32 away
    other.x = __shfl_xor_sync(0xffffffffu, raw.x, 4), other.y = __shfl_xor_sync(0xffffffffu, raw.y, 4);
    other.z = __shfl_xor_sync(0xffffffffu, raw.z, 4), other.w = __shfl_xor_sync(0xffffffffu, raw.w, 4);
    halves(other, far);
#pragma unroll
    for (int i = 0; i < 8; ++i) sin[i] = c < 4 ? -sin[i] : sin[i];
    if (a.key_norm == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * cos[i] + far[i] * sin[i];
        return;
    }
    double part[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i & 1] = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), part[i & 1]);
    double sum = part[0] + part[1];
#pragma unroll
    for (int offset = 1; offset < 8; offset <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    const double inverse = rsqrt(sum * (1.0 / kDim) + a.eps);
    const __half *norm = a.key_norm + static_cast<int64_t>(a.layer_begin + layer) * kDim;
    float own[8], its[8];
    halves(*reinterpret_cast<const uint4 *>(norm + 8 * c), own);
    halves(*reinterpret_cast<const uint4 *>(norm + 8 * (c ^ 4)), its);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double x = v[i] * inverse * static_cast<double>(own[i]), y = far[i] * inverse * static_cast<double>(its[i]);
        v[i] = static_cast<float>(x * static_cast<double>(cos[i]) + y * static_cast<double>(sin[i]));
    }
}

// Bound by latency up to a few hundred tokens: 1 token 1.6 us, 2047 tokens 2.4, in two layers 3.8;
// with queries to FP32 75 tokens 1.9, 1024 tokens 4.5, 2047 tokens 8.1 (29 MB, 4.5 at the copy rate).
__global__ void __launch_bounds__(kThreads) int4_append_kernel(const __grid_constant__ AppendArgs a) {
    pkv::pdl_wait();
    pkv::pdl_launch_dependents();
    const int layer = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (static_cast<int>(blockIdx.x) >= a.tile_ctas) {
        rotate_queries(a, layer, (static_cast<int>(blockIdx.x) - a.tile_ctas) * kQuerySpan, warp, lane);
        return;
    }
    // Lane c of a row's eight: dims 8 c .. + 7 of one token's K or V head.
    const int c = lane & 7, head = warp & 3;
    const bool is_key = warp < kHeads;
    const int token = static_cast<int>(blockIdx.x) * kSpan + (lane >> 3);
    const bool listed = token < a.tokens;
    const int64_t from = layer * a.layer_stride + min(token, a.tokens - 1) * a.token_stride + head * kDim + 8 * c;
    const uint4 raw = *reinterpret_cast<const uint4 *>((is_key ? a.key : a.value) + from);
    const int slot = listed ? a.slots[token] : -1;
    const bool ok = slot >= 0 && slot < static_cast<int64_t>(a.cache.num_blocks) * kSlots;
    if (listed && !ok && c == 0 && warp == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
    float v[8];
    halves(raw, v);
    if (is_key && a.rope != nullptr) turn_chunk(a, layer, ok ? checked_position(a, token) : 0, c, raw, v);
    uint32_t word, scale;
    pkv::int4::encode_chunk(v, word, scale);
    if (!ok) return;
    uint8_t *const to = pkv::int4::block_at(a.cache, a.layer_begin + layer, slot / kSlots) + head * pkv::int4::kHeadBytes;
    if (is_key) pkv::int4::store_key(to, c, slot % kSlots, word, scale);
    else pkv::int4::store_value(to, c, slot % kSlots, word, scale);
}

// K and V of `blocks` as FP16, each [i][slot][head][dim].  One CTA per block, a word of codes a
// thread: 16 consecutive bytes out, a warp whole rows (a thread with a group of 32 bytes filled
// half of each sector at a time: 256 blocks 4.9 us instead of 2.7, 4.2 MB out and 1.2 in).  Bound by
// latency: of the launch and of an id, codes and scales read one after the other; 1 block takes 1.5
// us.  index_out (nullable) receives 0 .. count - 1, the block table of the outputs as a pool.
constexpr int kReadThreads = kSlots * kHeads * 8;
constexpr int64_t kBlockValues = kSlots * kHeads * kDim;

__device__ __forceinline__ uint4 decode_word(uint32_t word, uint32_t scale) {
    const __half2 s = __half2half2(__ushort_as_half(static_cast<unsigned short>(scale << 7)));
    const uint32_t swapped = pkv::int4::swap_bytes(word);
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 n = pkv::int4::nibble_pair(word, swapped, i);
        v[i] = pkv::pack_half2(__hmul2(__hsub2(n, __float2half2_rn(i & 1 ? 24.f : 264.f)), s));  // exact
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__global__ void __launch_bounds__(kReadThreads)
    int4_read_kernel(const pkv::int4::Cache cache, int layer, const int32_t *blocks, __half *key_out, __half *value_out,
                     int32_t *index_out, int32_t *error_flag) {
    pkv::pdl_launch_dependents();
    pkv::pdl_wait();
    const int block = blocks[blockIdx.x];
    const bool bad = block < 0 || block >= cache.num_blocks;
    if (bad && threadIdx.x == 0) atomicOr(error_flag, PKV_DEVICE_BAD_BLOCK);
    if (index_out != nullptr && threadIdx.x == 0) index_out[blockIdx.x] = blockIdx.x;
    const int c = threadIdx.x & 7, head = (threadIdx.x >> 3) & 3, token = threadIdx.x >> 5;
    uint32_t k = 0, v = 0, ks = 0, vs = 0;
    if (!bad) {
        const uint8_t *from = pkv::int4::block_at(cache, layer, block) + head * pkv::int4::kHeadBytes;
        k = *reinterpret_cast<const uint32_t *>(from + pkv::int4::key_words(c >> 1, token) + 4 * (c & 1));
        v = *reinterpret_cast<const uint32_t *>(from + pkv::int4::value_word(c, token));
        ks = from[pkv::int4::scale_at(pkv::int4::kKeyScaleAt, c >> 1, token)];
        vs = from[pkv::int4::scale_at(pkv::int4::kValueScaleAt, c >> 1, token)];
    }
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (kBlockValues / 8) + threadIdx.x;
    reinterpret_cast<uint4 *>(key_out)[at] = decode_word(k, ks);
    reinterpret_cast<uint4 *>(value_out)[at] = decode_word(v, vs);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

namespace pkv::int4 {

int check_cache(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer_begin, int32_t layer_count) {
    if (storage == nullptr || !aligned16(storage)) {
        return fail(PKV_VALUE_ERROR, "int4 cache: the storage is required and must be 16-byte aligned");
    }
    if (layers < 1 || num_blocks < 1 || num_blocks > INT32_MAX / PKV_BLOCK_TOKENS) {
        return fail(PKV_VALUE_ERROR, "int4 cache: layer or block count out of range");
    }
    if (layer_begin < 0 || layer_count < 1 || layer_count > layers - layer_begin) {
        return fail(PKV_VALUE_ERROR, "int4 cache: layers out of range");
    }
    return PKV_OK;
}

}  // namespace pkv::int4

extern "C" int pkv_int4_append_kv(void *storage, int32_t layers, int32_t num_blocks, int32_t layer_begin,
                                  int32_t layer_count, const void *key, const void *value, int64_t src_layer_stride,
                                  int64_t src_token_stride, const int32_t *slots, const int32_t *positions,
                                  int32_t tokens, const void *rope_table, const void *query_norm, const void *key_norm,
                                  double eps, const void *query_in, int64_t q_layer_stride, int64_t q_token_stride,
                                  void *query_out, int32_t query_out_fp32, int64_t q_out_layer_stride,
                                  int64_t q_out_token_stride, int32_t *error_flag, void *stream) {
    pkv::clear_error();
    const int rc = pkv::int4::check_cache(storage, layers, num_blocks, layer_begin, layer_count);
    if (rc) return rc;
    if (key == nullptr || value == nullptr || slots == nullptr || error_flag == nullptr || tokens < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 append: key, value, slots and error_flag are required");
    }
    if ((rope_table != nullptr) != (positions != nullptr) || (query_in != nullptr) != (query_out != nullptr) ||
        (query_in != nullptr && rope_table == nullptr)) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 append: rope_table goes with positions, query with both and an output");
    }
    if ((query_norm != nullptr) != (key_norm != nullptr) || (key_norm != nullptr && rope_table == nullptr)) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 append: the norms go together and with rope_table");
    }
    if (!aligned16(key) || !aligned16(value) || src_layer_stride % 8 || src_token_stride % 8 || !aligned16(rope_table) ||
        !aligned16(query_norm) || !aligned16(key_norm) ||
        (query_in && (!aligned16(query_in) || !aligned16(query_out) || q_layer_stride % 8 || q_token_stride % 8 ||
                      q_out_layer_stride % 8 || q_out_token_stride % 8))) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 append: rows must be 16-byte aligned with strides in multiples of 8");
    }
    if (tokens > pkv::int4::kMostEntries) return pkv::fail(PKV_VALUE_ERROR, "int4 append: too many tokens");
    if (layer_count > 65535) return pkv::fail(PKV_VALUE_ERROR, "int4 append: layers out of range");
    if (tokens == 0) return PKV_OK;
    AppendArgs a = {};
    a.cache = pkv::int4::cache_of(storage, layers, num_blocks);
    a.layer_begin = layer_begin;
    a.key = static_cast<const __half *>(key);
    a.value = static_cast<const __half *>(value);
    a.layer_stride = src_layer_stride;
    a.token_stride = src_token_stride;
    a.slots = slots;
    a.positions = positions;
    a.tokens = tokens;
    a.rope = static_cast<const __half *>(rope_table);
    a.query_norm = static_cast<const __half *>(query_norm);
    a.key_norm = static_cast<const __half *>(key_norm);
    a.eps = eps;
    a.query_in = static_cast<const __half *>(query_in);
    a.query_out = query_out;
    a.query_out_fp32 = query_out_fp32;
    a.q_layer_stride = q_layer_stride;
    a.q_token_stride = q_token_stride;
    a.q_out_layer_stride = q_out_layer_stride;
    a.q_out_token_stride = q_out_token_stride;
    a.error_flag = error_flag;
    a.tile_ctas = (tokens + kSpan - 1) / kSpan;
    const dim3 grid(a.tile_ctas + (query_in != nullptr ? (tokens + kQuerySpan - 1) / kQuerySpan : 0), layer_count);
    const cudaError_t e =
        pkv::launch_pdl(int4_append_kernel, grid, dim3(kThreads), static_cast<cudaStream_t>(stream), a);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 append launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

namespace {

int read_blocks(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer, const int32_t *blocks,
                int32_t count, void *key_out, void *value_out, int32_t *index_out, int32_t *error_flag, void *stream) {
    const int rc = pkv::int4::check_cache(storage, layers, num_blocks, layer, 1);
    if (rc) return rc;
    if (blocks == nullptr || key_out == nullptr || value_out == nullptr || error_flag == nullptr || count < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 read: blocks, outputs and error_flag are required");
    }
    if (!aligned16(key_out) || !aligned16(value_out)) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 read: the outputs must be 16-byte aligned");
    }
    if (count == 0) return PKV_OK;
    const cudaError_t e = pkv::launch_pdl(int4_read_kernel, dim3(count), dim3(kReadThreads), static_cast<cudaStream_t>(stream),
                                          pkv::int4::cache_of(storage, layers, num_blocks), layer, blocks,
                                          static_cast<__half *>(key_out), static_cast<__half *>(value_out), index_out,
                                          error_flag);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 read launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

}  // namespace

extern "C" int pkv_int4_read_blocks(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer,
                                    const int32_t *blocks, int32_t count, void *key_out, void *value_out,
                                    int32_t *error_flag, void *stream) {
    pkv::clear_error();
    return read_blocks(storage, layers, num_blocks, layer, blocks, count, key_out, value_out, nullptr, error_flag, stream);
}

// Two ways to attend to a prompt chunk.
//
// By tiles: the request's blocks become an FP16 pool of one layer in the workspace (the values
// are FP16 numbers: nothing is rounded), which the tensor-core prompt kernel attends to; that
// kernel reads every block once for each 16 queries, and a tile's keys one after another, in several
// parts where there are few tiles.
//
// By rows: each token a row of the decode attention, which cuts the keys over the whole GPU but
// reads a row's blocks for each token.  For a few tokens behind a long context.
namespace {

// Rows take about 6.5 us and 1.2 ns for each block of each row, tiles 7 us and 0.87 us for each 64
// keys that the last tile walks, where its keys are not cut into parts: 600 blocks a step is where
// they meet, and 7500 blocks with parts (3 tokens behind 1900 take 8.4 us by rows and 16 by tiles, 75
// behind 601 11.7 and 14.3, 150 behind 256 11.9 and 12.6, 110 behind 1000 16.7 and 18.0, 150 behind
// 1000 19.8 and 18.1, 220 behind 256 15.3 and 13.6).  At the beginning it is short rows, a piece each,
// against the first tiles: 16 tokens 6.4 and 7.4 us, 75 tokens 8.0 and 8.3, 110 tokens 10.3 and 8.7.
bool by_rows(int start, int tokens) {
    const int64_t blocks = static_cast<int64_t>(tokens) * (start + tokens / 2) / kSlots;
    if (start < 64) return tokens <= 80 && start + tokens <= 8 * kSlots;
    return blocks < 7500 && blocks < 600 * ((start + tokens) / 64);
}

// Of the tiles: an FP16 pool of one layer, its table, the partial results.
struct TilesWorkspace {
    int blocks, splits;
    int64_t table_at, partials_at, bytes;
};

int tiles_workspace(int device, int start, int tokens, TilesWorkspace *w) {
    if (const int rc = pkv::prefill_splits(device, start, tokens, &w->splits)) return rc;
    w->blocks = (start + tokens + kSlots - 1) / kSlots;
    w->table_at = static_cast<int64_t>(w->blocks) * 2 * kBlockValues * 2;
    w->bytes = w->table_at + static_cast<int64_t>(w->blocks) * 4;
    w->partials_at = (w->bytes + 15) / 16 * 16;
    const int64_t partials = pkv::prefill_splits_bytes(tokens, w->splits);
    if (partials > 0) w->bytes = w->partials_at + partials;
    return PKV_OK;
}

int check_chunk(int32_t start, int32_t tokens) {
    if (tokens < 1 || start < 0 || static_cast<int64_t>(start) + tokens > PKV_CONTEXT_LIMIT) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: the chunk must hold 1 or more tokens at positions below 2048");
    }
    return PKV_OK;
}

}  // namespace

extern "C" int pkv_int4_prefill_plan(int32_t device, int32_t start, int32_t tokens, int64_t *out_workspace_bytes) {
    pkv::clear_error();
    if (out_workspace_bytes == nullptr) return pkv::fail(PKV_VALUE_ERROR, "prefill plan: null pointer argument");
    if (const int rc = check_chunk(start, tokens)) return rc;
    if (by_rows(start, tokens)) return pkv::int4::rows_workspace(device, start, tokens, out_workspace_bytes);
    TilesWorkspace tiles;
    if (const int rc = tiles_workspace(device, start, tokens, &tiles)) return rc;
    *out_workspace_bytes = tiles.bytes;
    return PKV_OK;
}

extern "C" int pkv_int4_prefill_attention(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer,
                                          const void *query, int32_t query_fp32, int64_t query_stride,
                                          const int32_t *blocks, int32_t start, int32_t tokens, void *out,
                                          int64_t out_stride, void *workspace, int64_t workspace_bytes,
                                          int32_t *error_flag, void *stream) {
    pkv::clear_error();
    if (query == nullptr || blocks == nullptr || out == nullptr || error_flag == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: null pointer argument");
    }
    if (const int rc = check_chunk(start, tokens)) return rc;
    constexpr int64_t kRow = PKV_QUERY_HEADS * PKV_HEAD_DIM;
    if (!aligned16(query) || !aligned16(out) || query_stride % 8 || out_stride % 8 || query_stride < kRow ||
        out_stride < kRow) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: rows must be 16-byte aligned, 2048 or more values apart in multiples of 8");
    }
    if (by_rows(start, tokens)) {
        const int rc = pkv::int4::check_cache(storage, layers, num_blocks, layer, 1);
        if (rc) return rc;
        return pkv::int4::attend_rows(pkv::int4::cache_of(storage, layers, num_blocks), layer, query, query_fp32 != 0,
                                      query_stride, blocks, start, tokens, out, out_stride, workspace, workspace_bytes,
                                      error_flag, static_cast<cudaStream_t>(stream));
    }
    int device = 0;
    if (start > 0) {  // (at the beginning the plan asks for no device)
        const cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
    }
    TilesWorkspace tiles;
    if (const int rc = tiles_workspace(device, start, tokens, &tiles)) return rc;
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < tiles.bytes) {
        return pkv::fail(PKV_VALUE_ERROR, "prefill attention: the workspace is too small (see pkv_int4_prefill_plan)");
    }
    uint8_t *const base = static_cast<uint8_t *>(workspace);
    int32_t *const table = reinterpret_cast<int32_t *>(base + tiles.table_at);
    const int rc = read_blocks(storage, layers, num_blocks, layer, blocks, tiles.blocks, workspace,
                               static_cast<__half *>(workspace) + tiles.blocks * kBlockValues, table, error_flag, stream);
    if (rc) return rc;
    return pkv::launch_prefill_attention_tc(workspace, tiles.blocks, 0, query, query_fp32 != 0, true, query_stride, table,
                                            start, tokens, out, out_stride, error_flag, static_cast<cudaStream_t>(stream),
                                            tiles.splits,
                                            tiles.splits > 1 ? reinterpret_cast<float *>(base + tiles.partials_at) : nullptr);
}
