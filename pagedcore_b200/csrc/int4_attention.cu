// Batched one-token attention over the 4-bit KV cache (numbers and layout: int4.cuh):
//   out[b, h] = sum_t softmax_t(q[b, h] . K[t, h / 8] / 8) V[t, h / 8]
// over the lengths[b] tokens that row b's block table lists; for a decode layer the row's new
// token is written first, its K and the row's queries normed (where asked for) and rotated here.
//
// Work split: the batch's block tables form one flat list, CTA g streams piece g of it (three CTAs
// an SM): a producer warp copies whole blocks, 4608 consecutive bytes, into a ring, and warp w
// serves KV head w and its eight query heads from it.  A row that one piece holds is written
// directly; the others leave (m, l, O) partials at index row + piece (unique: along the pieces the
// pairs form a monotone staircase) that a second kernel merges.  A decode layer's new token is
// written by the warps of the piece that holds its row's last block, which also put it into their
// copy of that block: the copy may have been taken before the write.
//
// Math: mma.sync m16n8k16 on FP16 operands made from codes in registers (the values are FP16
// numbers), FP32 sums:
//   S^T[16 tok x 8 heads]  = K[16 x 64] . Q^T[64 x 8]
//   O^T[64 dims x 8 heads] += V^T[64 x 16] . P^T[16 x 8]
// The summed indices may be taken in any order, so a lane (g, t) reads 16 consecutive bytes
// of each: K of tokens 2 g and 2 g + 1 in dims 16 t .. + 15, which are one group, and V of
// tokens 4 t .. 4 t + 3 in dims 8 g .. + 7.  Rows g and g + 8 of the first product are tokens
// 2 g and 2 g + 1; two 8 x 8 transposes turn it into the second's operand, whose pairs of
// summed indices are then tokens 4 t, 4 t + 2 and 4 t + 1, 4 t + 3.
//
// Values go into the MMAs times 2^-6, so that 264 scales stay inside FP16 (256 + n times s
// minus 264 s is one rounding, exact); the factor of the scores and the last product undo it.
// Weights and the layer's queries go in as two FP16 numbers each, hi = x to 11 bits and
// lo = fp16(x - hi), at most 2^-21 of x off (one alone shows in the output beside its own
// rounding), below FP16's normal numbers 2^-24 (of a weight 2^-35 of the row's largest); a query
// head is scaled by the power of two that brings its largest value to 2^14 .. 2^15 first,
// whatever its range.  Scores, references, normaliser and sums are FP32.
//
// The softmax's reference is raised only when a weight would pass 2^15, and then to 2^11 below the
// largest score, so that most blocks touch neither it nor the sums; a row's weights are relative to
// one another whatever it is.
//
// What bounds it: 256 rows of 1 to 2048 tokens (16,500 blocks, 76 MB) take 25 us, 11.7 of them at
// the copy rate.  A (block, head) is 183 instructions, 266 clocks of its SM's quarter: 12 MMAs at 8
// clocks, 48 FP16 operations at 2 and about 24 FP32 ones, 216 in all, for timed together they take as
// long as one after the other.  (No counter shows a full pipe: over the whole kernel ALU 43 %, FMA
// 32 %, tensor 27 %, issue slots 52 %.)  The rest, about 9 us, is fixed: 3.4 to the first data, 3.4
// between an SM's first and last CTA, the merge.  (tcgen05 would read V from shared memory as FP16:
// 488 bytes a token and head there and back, 14 us of the 16.5 that the stream takes now.)

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <initializer_list>
#include <string>

#include "block_list.cuh"
#include "int4.cuh"
#include "pdl.h"
#include "ptx.cuh"
#include "status.h"

namespace {

using pkv::advance_row, pkv::load_rows, pkv::max8, pkv::Merge, pkv::out_of_order, pkv::Rows, pkv::sum8, pkv::total_blocks;

constexpr int kDim = PKV_HEAD_DIM;
constexpr int kHeads = PKV_KV_HEADS;
constexpr int kQueryHeads = PKV_QUERY_HEADS;
constexpr int kHeadGroup = kQueryHeads / kHeads;
constexpr int kSlots = PKV_BLOCK_TOKENS;
constexpr int kWarps = kHeads;     // consumers, one per KV head
constexpr int kProducer = kWarps;  // the warp that fills the ring
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kChunk = 4;  // blocks per stage, and the least of a piece
constexpr int kStages = 2;
constexpr int kStageBytes = kChunk * pkv::int4::kBlockBytes;
constexpr int kFreshBytes = 80;  // of a row's new token in one head, see write_new
constexpr int kFreshOk = 72;
constexpr int kFreshAt = kStages * kStageBytes;
constexpr int kSmem = kFreshAt + kWarps * kFreshBytes;
constexpr uint32_t kWaitPolls = 1u << 24;
constexpr int kRowCost = 3;  // below a chunk's blocks
constexpr int kWeighedRows = 256;
constexpr int kMostGrid = 65535;
static_assert(static_cast<int64_t>(kMostGrid) * kThreads < INT32_MAX - pkv::int4::kMostRows, "a row loop steps past 32 bits");
constexpr int kShortRow = 8;
static_assert(kRowCost < kChunk, "a piece could lie in the cost of one row");  // pieces are kRowCost + 1 long or more
constexpr float kScaleLog2 = 0.125f * 1.4426950408889634f;  // 64^-0.5 * log2(e)
constexpr float kValueFactor = 0x1p-6f;  // of the values in the MMAs
constexpr float kMostWeight = 15.0f;  // log2 of the largest weight
constexpr float kWeightShift = 11.0f;  // ... and of one at the reference when that is set
constexpr float kFarScore = 0x1p20f;
constexpr float kLowest = -FLT_MAX;  // no finite score is below
constexpr int kPartial = kQueryHeads * (kDim + 2);  // floats of a partial

// What the rows are: sequences with rotated FP16 queries; sequences with a new token each (a
// decode layer), whose queries are normed and rotated here; or the tokens of a prompt chunk, with
// rotated FP16 or FP32 queries: token t is a row of start + t + 1 tokens over the first blocks of
// the request's table.
enum class Kind { kPlain, kFresh, kChunk };

// Blocks of a chunk's rows before row r.
__host__ __device__ __forceinline__ int blocks_before(int start, int r) {
    const auto upto = [](int n) { return n + kSlots * (n / kSlots) * (n / kSlots - 1) / 2 + n / kSlots * (n % kSlots); };
    return upto(start + r) - upto(start);
}

struct Args {
    pkv::int4::Cache cache;
    int32_t layer;
    const __half *query;
    const float *query32;  // of a chunk, in place of query where it is not null
    int64_t query_stride;
    const __half *key;  // the new tokens, with rope; null for the attention alone
    const __half *value;
    int64_t kv_stride;
    const __half *rope;
    const __half *query_norm;  // of this layer, or null
    const __half *key_norm;
    double eps;
    const int32_t *lengths;  // null for a chunk
    const int32_t *prefix;   // null for a chunk
    const int32_t *flat;     // of a chunk the request's table
    int32_t start;           // of a chunk
    int32_t batch;
    int32_t capacity;  // of flat; the batch's blocks are prefix[batch]
    int32_t grid;
    int32_t clear;     // rows without blocks give zeros (else they are left alone)
    __half *out;
    int64_t out_stride;
    float *part_o;   // [batch + grid][32][64]
    float *part_ml;  // [batch + grid][32][2]
    int32_t *error_flag;
};

// The arguments with the tables that the kind of rows has.
template <Kind R>
struct ArgsOf : Args {
    explicit ArgsOf(const Args &args) : Args(args) {}

    __device__ __forceinline__ int prefix_at(int row) const {
        return R == Kind::kChunk ? blocks_before(start, row) : prefix[row];
    }
    __device__ __forceinline__ int length_at(int row) const { return R == Kind::kChunk ? start + row + 1 : lengths[row]; }
};

// Most pieces of a list of `total` blocks in `rows` rows with blocks: one per CTA, and one per
// chunk or per row, whichever are more.  (A captured launch has a CTA for every resident slot.)
__host__ __device__ __forceinline__ int pieces_of(int total, int rows, int grid) {
    const int chunks = (total + kChunk - 1) / kChunk, rows_most = rows < total ? rows : total;
    const int most = chunks > rows_most ? chunks : rows_most;
    return most < 1 ? 1 : most < grid ? most : grid;
}

// The rows of a list of up to kWeighedRows rows, 32 k + lane in each lane; what they list before
// block 0 (of a list that is out of order) is left out, so that a row found ends past its block.
struct RowScan {
    static constexpr int kParts = kWeighedRows / 32;
    int first[kParts], last[kParts];
    unsigned held[kParts];  // rows with blocks
    int count;    // ... how many
    bool short_rows;  // none has more than kShortRow

    template <Kind R>
    __device__ __forceinline__ RowScan(const ArgsOf<R> &a, int lane) {
        bool long_row = false;
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            const int r = 32 * k + lane;
            first[k] = last[k] = 0;
            if (r < a.batch) first[k] = max(a.prefix_at(r), 0), last[k] = a.prefix_at(r + 1);
            long_row |= last[k] > first[k] && last[k] - first[k] > kShortRow;
        }
        short_rows = !__any_sync(0xffffffffu, long_row);
        count = 0;
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            held[k] = __ballot_sync(0xffffffffu, last[k] > first[k]);
            count += __popc(held[k]);
        }
    }
    // Rows with blocks up to row `row`.
    __device__ __forceinline__ int rank(int row) const {
        int upto = 0;
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            const int n = row - 32 * k;  // the last row of this part that counts
            if (n >= 0) upto += __popc(n >= 31 ? held[k] : held[k] & ((2u << n) - 1u));
        }
        return upto;
    }
    // The first block of weight `target` or more, and its row, which ends past it in any list;
    // `total` where there is none.
    __device__ __forceinline__ int block_at(uint32_t target, int total, int lane, int &row) const {
        int before = 0;
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            const uint32_t cost = kRowCost * (before + __popc(held[k] & ((2u << lane) - 1u)));
            const unsigned found = __ballot_sync(0xffffffffu, last[k] > first[k] && last[k] - 1 + cost >= target);
            if (found != 0) {
                const int from = __ffs(found) - 1;
                row = 32 * k + from;
                const int block = max(first[k], target > cost ? static_cast<int>(target - cost) : 0);
                return __shfl_sync(0xffffffffu, min(block, total), from);
            }
            before += __popc(held[k]);
        }
        row = INT32_MAX;
        return total;
    }
    // Where the `index`-th row with blocks begins and ends, cut at `total`, and the row.  (With an exit
    // per part, as above, the rows of both searches land in local memory: 0.6 us a call.)
    __device__ __forceinline__ void row_at(int index, int total, int lane, int &begin, int &end, int &row) const {
        int found = INT32_MAX, from = 0, to = 0;
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            if (last[k] > first[k] && __popc(held[k] & ((1u << lane) - 1u)) == index) found = 32 * k + lane, from = first[k], to = last[k];
            index -= __popc(held[k]);
        }
        row = __reduce_min_sync(0xffffffffu, found);
        begin = min(__shfl_sync(0xffffffffu, from, row & 31), total);
        end = row == INT32_MAX ? begin : min(__shfl_sync(0xffffffffu, to, row & 31), total);
    }
};

// How the list is cut.  Short rows (kShortRow blocks or less, a CTA for each): one piece a row.
// Else a block weighs 1 and a row's first block kRowCost more, what it costs a CTA to begin a row
// (its queries, its result); piece g holds the blocks whose weights, summed to and without the
// block itself, lie in [g, g + 1) * weight / pieces.  A piece is kRowCost + 1 long or more, so none
// is without blocks.  Beyond kWeighedRows rows, where a CTA has several rows and they even out, rows
// weigh nothing.  (A decode layer of 256 rows of 1 to 2048 tokens takes 34.0, 33.2, 32.3 and 32.0 us
// with a cost of 0, 1, 2 and 3.  Pieces of a chunk or more made short rows wait for one another: 8
// rows of 5 tokens took 8.7 us and their layer with norms 16.3, a piece each 3.3 and 5.2.)
struct Cut {
    int total, pieces;
    bool by_row;
    uint32_t weight, whole, rest;  // weight = whole * pieces + rest

    template <Kind R>
    __device__ __forceinline__ Cut(const ArgsOf<R> &a, int rows_with_blocks, bool short_rows) {
        total = total_blocks(a);
        by_row = short_rows && rows_with_blocks > 0 && rows_with_blocks <= a.grid;
        pieces = by_row ? rows_with_blocks : pieces_of(total, a.batch <= kWeighedRows ? rows_with_blocks : total, a.grid);
        weight = static_cast<uint32_t>(total) + kRowCost * rows_with_blocks;
        whole = weight / pieces;
        rest = weight % pieces;
    }
    // Of block `block` in the list's `rank`-th row with blocks (counted from 1).
    __device__ __forceinline__ int piece_of(int block, int rank) const {
        return by_row ? rank - 1 : static_cast<int>((static_cast<int64_t>(block) + kRowCost * rank) * pieces / weight);
    }
    // The least weight that is in piece g, g <= pieces.  (No product passes 32 bits, for pieces <=
    // kMostGrid: divisions of 64 bits cost a small call 0.2 us.)
    __device__ __forceinline__ uint32_t begins(int g) const {
        return whole * g + (rest * g + pieces - 1) / static_cast<uint32_t>(pieces);
    }
};

// D = A(16x16, row) * B(16x8, col) + D, FP16 operands.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack(__half2 h) { return pkv::pack_half2(h); }

__device__ __forceinline__ __half2 as_half2(uint32_t bits) { return *reinterpret_cast<const __half2 *>(&bits); }

// A pair of scales, two FP16 numbers, ready for value_pair: times 2^-6, and the products that
// take 16 + 8 and 256 + 8 away.
struct Steps {
    __half2 step, low, high;
    __device__ __forceinline__ explicit Steps(uint32_t scales) {
        const __half2 s = as_half2(scales);
        step = __hmul2(s, __float2half2_rn(kValueFactor));
        low = __hmul2(s, __float2half2_rn(-24.f * kValueFactor));
        high = __hmul2(s, __float2half2_rn(-264.f * kValueFactor));
    }
};

// Codes i of both halves of a word as values times 2^-6.
__device__ __forceinline__ uint32_t value_pair(uint32_t word, uint32_t swapped, int i, const Steps &s) {
    return pack(__hfma2(pkv::int4::nibble_pair(word, swapped, i), s.step, i & 1 ? s.low : s.high));
}

// A lane's 16 query dims (16 t .. + 15) of head g of its warp, as MMA operands.
struct Query {
    uint32_t high[8], low[8];
    float factor0, factor1;  // of the scores of heads 2 t and 2 t + 1

    template <Kind R>
    __device__ __forceinline__ void load(const Args &a, int row, int length, int warp, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const int64_t at = row * a.query_stride + (warp * kHeadGroup + g) * kDim;
        if constexpr (R == Kind::kPlain) {
            const uint4 *from = reinterpret_cast<const uint4 *>(a.query + at + 16 * t);
            const uint4 x = from[0], y = from[1];
            high[0] = x.x, high[1] = x.y, high[2] = x.z, high[3] = x.w;
            high[4] = y.x, high[5] = y.y, high[6] = y.z, high[7] = y.w;
            factor0 = factor1 = kScaleLog2 / kValueFactor;
            return;
        }
        float q[16];
        if constexpr (R == Kind::kFresh) {
            turn(a, a.query + at, length, t, q);
        } else if (a.query32 != nullptr) {
            const float4 *from = reinterpret_cast<const float4 *>(a.query32 + at + 16 * t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 v = from[i];
                q[4 * i] = v.x, q[4 * i + 1] = v.y, q[4 * i + 2] = v.z, q[4 * i + 3] = v.w;
            }
        } else {
            pkv::int4::load16(a.query + at + 16 * t, q);
        }
        halve(q, t);
    }

    // Norm (where there is one) and rotation of a head's dims, 16 t .. + 15 in each of its four lanes.
    static __device__ __forceinline__ void turn(const Args &a, const __half *src, int length, int t, float (&q)[16]) {
        float other[16], cos[16], sin[16];
        pkv::int4::load16(src + 16 * t, q);
        pkv::int4::load16(src + 16 * (t ^ 2), other);
        if (a.query_norm != nullptr) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(q[i], q[i], sum);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const float inverse = rsqrtf(sum * (1.f / kDim) + static_cast<float>(a.eps));
            pkv::int4::load16(a.query_norm + 16 * t, cos);
            pkv::int4::load16(a.query_norm + 16 * (t ^ 2), sin);
#pragma unroll
            for (int i = 0; i < 16; ++i) q[i] *= inverse * cos[i], other[i] *= inverse * sin[i];
        }
        const int position = length >= 1 && length <= PKV_CONTEXT_LIMIT ? length - 1 : 0;
        const __half *factors = a.rope + position * (kDim / 2) + 16 * (t & 1);
        pkv::int4::load16(factors, cos);
        pkv::int4::load16(factors + PKV_CONTEXT_LIMIT * (kDim / 2), sin);
#pragma unroll
        for (int i = 0; i < 16; ++i) q[i] = q[i] * cos[i] + (t < 2 ? -other[i] : other[i]) * sin[i];
    }

    // The head's values, scaled, as two FP16 numbers each.
    __device__ __forceinline__ void halve(const float (&q)[16], int t) {
        float largest = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (fabsf(q[i]) < INFINITY) largest = fmaxf(largest, fabsf(q[i]));
        }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const int e = max((__float_as_int(largest) >> 23) - 127 - 14, -100);  // zeros and FP32's subnormals: 2^100
        const float scale = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = q[2 * i] * scale, y = q[2 * i + 1] * scale;
            const __half2 h = __floats2half2_rn(x, y);
            const float2 f = __half22float2(h);
            high[i] = pack(h);
            low[i] = pack(__floats2half2_rn(x - f.x, y - f.y));
        }
        const float factor = __int_as_float((127 + e) << 23) * (kScaleLog2 / kValueFactor);
        factor0 = __shfl_sync(0xffffffffu, factor, 8 * t);
        factor1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
    }
};

// A head's queries of a row into L1.
template <Kind R>
__device__ __forceinline__ void prefetch_query(const Args &a, int row, int warp, int lane) {
    const int64_t at = row * a.query_stride + warp * kHeadGroup * kDim + lane * 16;
    if (R == Kind::kChunk && a.query32 != nullptr) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.query32 + at));
    else asm volatile("prefetch.global.L1 [%0];" ::"l"(a.query + at));
}

// Copies of memory that one CTA reads once.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy)
        : "memory");
}

__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity) {
    return pkv::mbar_test_wait(bar, parity) || pkv::mbar_wait_bounded(bar, parity, kWaitPolls);
}

// What a block id outside the cache reads as.
__device__ __align__(16) const uint8_t kZeroBlock[pkv::int4::kBlockBytes] = {};

// The new token of row `row` into its slot of `block`, one head a warp, and into the warp's 80
// bytes of shared memory at `fresh`: 32 of K codes, 32 of V codes, 4 + 4 scales, and whether there
// is one.
__device__ __forceinline__ void write_new(const Args &a, int row, int length, int block, int warp, int lane, uint8_t *fresh) {
    const bool in_range = length >= 1 && length <= PKV_CONTEXT_LIMIT;
    const bool ok = in_range && block >= 0 && block < a.cache.num_blocks;
    const int64_t from = row * a.kv_stride + warp * kDim + 2 * lane;
    const __half2 k = *reinterpret_cast<const __half2 *>(a.key + from), v = *reinterpret_cast<const __half2 *>(a.value + from);
    const pkv::int4::KeyTurn turn(a.key_norm, a.rope, in_range ? length - 1 : 0, lane);
    const float2 key = a.key_norm != nullptr ? pkv::int4::turn_key<true>(k, turn, a.eps) : pkv::int4::turn_key<false>(k, turn, a.eps);
    const float2 value = __half22float2(v);
    uint32_t key_word, key_scale, value_word, value_scale;
    pkv::int4::encode_pair(key.x, key.y, lane, key_word, key_scale);
    pkv::int4::encode_pair(value.x, value.y, lane, value_word, value_scale);
    if (lane % 4 == 0) {
        reinterpret_cast<uint32_t *>(fresh)[lane >> 2] = key_word;
        reinterpret_cast<uint32_t *>(fresh)[8 + (lane >> 2)] = value_word;
    }
    if (lane % 8 == 0) {
        fresh[64 + (lane >> 3)] = static_cast<uint8_t>(key_scale);
        fresh[68 + (lane >> 3)] = static_cast<uint8_t>(value_scale);
    }
    if (lane == 0) *reinterpret_cast<int *>(fresh + kFreshOk) = ok;
    if (ok) {
        uint8_t *const to = pkv::int4::block_at(a.cache, a.layer, block) + warp * pkv::int4::kHeadBytes;
        const int slot = (length - 1) % kSlots;
        if (lane % 4 == 0) {
            pkv::int4::store_key(to, lane >> 2, slot, key_word, key_scale);
            pkv::int4::store_value(to, lane >> 2, slot, value_word, value_scale);
        }
    } else if (warp == 0 && lane == 0) {
        atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK | (in_range ? 0 : PKV_DEVICE_BAD_POSITION));
    }
    __syncwarp();
}

// The same token into the copy of its (block, head) at `head` in shared memory.
__device__ __forceinline__ void put_fresh(const uint8_t *fresh, uint8_t *head, int slot, int lane) {
    if (*reinterpret_cast<const int *>(fresh + kFreshOk) == 0) return;
    if (lane < 8) {
        *reinterpret_cast<uint32_t *>(head + pkv::int4::key_words(lane >> 1, slot) + 4 * (lane & 1)) =
            reinterpret_cast<const uint32_t *>(fresh)[lane];
    } else if (lane < 16) {
        *reinterpret_cast<uint32_t *>(head + pkv::int4::value_word(lane - 8, slot)) = reinterpret_cast<const uint32_t *>(fresh)[lane];
    } else if (lane < 24) {
        const int first = lane < 20 ? pkv::int4::kKeyScaleAt : pkv::int4::kValueScaleAt;
        head[pkv::int4::scale_at(first, lane & 3, slot)] = fresh[64 + lane - 16];
    }
    __syncwarp();
}

// The producer warp: copies the blocks of [begin, end) chunk by chunk, a chunk ending with its
// row.
template <Kind R>
__device__ __forceinline__ void fill_ring(const ArgsOf<R> &a, int begin, int end, int row, int lane, uint8_t *smem,
                                          uint64_t *full, uint64_t *empty) {
    const uint64_t policy = pkv::l2_policy_evict_first();
    const uint32_t ring = pkv::smem_addr(smem);
    // The ids of the list's next 64 blocks, 32 at a time, a window ahead.
    // (Of a chunk, whose rows share one short table, each id when it is needed.)
    int ids_base = begin, ids = 0, ids_next = 0;
    if constexpr (R != Kind::kChunk) {
        if (begin + lane < end) ids = a.flat[begin + lane];
        if (begin + 32 + lane < end) ids_next = a.flat[begin + 32 + lane];
    }
    Rows rows = load_rows(a, row, lane);
    int row_end = __shfl_sync(0xffffffffu, rows.last, 0);
    int issued = 0;
    bool ok = true;
    for (int at = begin; at < end;) {
        if (at >= row_end) {
            row = advance_row(a, rows, row + 1, at, lane);
            if (row >= a.batch) break;  // prefix does not grow from row to row: the consumers stop here too
            row_end = __shfl_sync(0xffffffffu, rows.last, row - rows.base);
        }
        const int n = min(kChunk, min(row_end, end) - at);
        int block;  // of lane's copy
        if constexpr (R == Kind::kChunk) {
            const int row_first = __shfl_sync(0xffffffffu, rows.first, row - rows.base);
            block = a.flat[at - row_first + min(lane, n - 1)];
        } else {
            if (at - ids_base >= 32) {
                ids = ids_next;
                ids_base += 32;
                const int ahead = ids_base + 32 + lane;
                ids_next = ahead < end ? a.flat[ahead] : 0;
            }
            const int offset = at - ids_base + min(lane, n - 1);
            const int near = __shfl_sync(0xffffffffu, ids, offset & 31);
            const int far = __shfl_sync(0xffffffffu, ids_next, offset & 31);
            block = offset < 32 ? near : far;
        }
        const bool bad = block < 0 || block >= a.cache.num_blocks;  // reported, and read as zeros
        if (bad && lane < n) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        const int stage = issued % kStages;
        if (issued >= kStages) {
            ok = __all_sync(0xffffffffu, wait_bounded(pkv::smem_addr(&empty[stage]), (issued / kStages - 1) & 1));
            if (!ok) break;  // a consumer gave up
        }
        const uint32_t bar = pkv::smem_addr(&full[stage]);
        if (lane == 0) pkv::mbar_arrive_expect_tx(bar, n * pkv::int4::kBlockBytes);
        __syncwarp();
        if (lane < n) {
            bulk_load(ring + stage * kStageBytes + lane * pkv::int4::kBlockBytes,
                      bad ? kZeroBlock : pkv::int4::block_at(a.cache, a.layer, block), pkv::int4::kBlockBytes, bar, policy);
        }
        at += n;
        ++issued;
    }
    if (!ok && lane == 0) atomicOr(a.error_flag, PKV_DEVICE_WAIT_TIMEOUT);
    // No copy may land after the CTA has left.
    for (int c = max(0, issued - kStages); c < issued; ++c) {
        wait_bounded(pkv::smem_addr(&full[c % kStages]), (c / kStages) & 1);
    }
}

// a * b per lane, round to nearest.
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// One row's running softmax of heads 2 t and 2 t + 1, over the tokens of the lane's rows.
struct Sums {
    float m0, m1;  // the references: weights are 2^(score - m)
    uint64_t l;    // the normalisers, an FP32 pair
    float o[4][4];

    __device__ __forceinline__ void clear() {
        m0 = m1 = kLowest;
        l = 0;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
    }

    // log2 of the weights of products s.  The product is rounded by itself, as raise does: far
    // out, what a fused operation keeps of it would be large (2^-24 of 2^38, in the exponent).
    __device__ __forceinline__ void exponents(const float (&s)[4], const Query &q, float (&x)[4]) const {
        const uint64_t reference = pkv::f32x2(-m0, -m1);  // (a packed product would be fused with the sum)
        const uint64_t p = pkv::f32x2(__fmul_rn(s[0], q.factor0), __fmul_rn(s[1], q.factor1));
        const uint64_t r = pkv::f32x2(__fmul_rn(s[2], q.factor0), __fmul_rn(s[3], q.factor1));
        const float2 first = pkv::unpack_f32x2(pkv::add_f32x2(p, reference));
        const float2 second = pkv::unpack_f32x2(pkv::add_f32x2(r, reference));
        x[0] = first.x, x[1] = first.y, x[2] = second.x, x[3] = second.y;
    }

    // References for scores that reach top0 and top1 in this lane.
    __device__ __forceinline__ void raise(float top0, float top1) {
        top0 = max8(top0);
        top1 = max8(top1);
        // Far out, where the shift would soon be lost in its rounding, the maximum itself.
        top0 = fmaxf(m0, fabsf(top0) > kFarScore ? top0 : top0 - kWeightShift);
        top1 = fmaxf(m1, fabsf(top1) > kFarScore ? top1 : top1 - kWeightShift);
        const float alpha0 = pkv::exp2_approx(m0 - top0), alpha1 = pkv::exp2_approx(m1 - top1);
        m0 = top0;
        m1 = top1;
        l = mul_f32x2(l, pkv::f32x2(alpha0, alpha1));
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[mt][0] *= alpha0, o[mt][1] *= alpha1, o[mt][2] *= alpha0, o[mt][3] *= alpha1;
    }
};

// Where a lane reads its bytes of a (block, head), as shared memory addresses.
struct Places {
    uint32_t k, v, ks, vs;

    __device__ __forceinline__ Places(uint32_t head, int lane) {
        const int g = lane >> 2, t = lane & 3;
        k = head + pkv::int4::key_words(t, 2 * g);
        v = head + pkv::int4::kValueAt + lane * 16;
        ks = head + pkv::int4::scale_at(pkv::int4::kKeyScaleAt, t, 2 * g);
        vs = head + pkv::int4::scale_at(pkv::int4::kValueScaleAt, g >> 1, 4 * t);
    }

    __device__ __forceinline__ Places at(uint32_t bytes) const {
        Places p = *this;
        p.k += bytes, p.v += bytes, p.ks += bytes, p.vs += bytes;
        return p;
    }
};

struct Tile {
    uint4 k, v;
    uint32_t ks, vs;

    // Block BLOCK of the stage at `p`.
    template <int BLOCK>
    __device__ __forceinline__ void load(const Places &p) {
        constexpr int kAt = BLOCK * pkv::int4::kBlockBytes;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
                     : "=r"(k.x), "=r"(k.y), "=r"(k.z), "=r"(k.w) : "r"(p.k), "n"(kAt));
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p.v), "n"(kAt));
        asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=r"(ks) : "r"(p.ks), "n"(kAt));
        asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(vs) : "r"(p.vs), "n"(kAt));
    }
};

template <Kind R>
__device__ __forceinline__ void score(const Tile &tile, const Query &q, float (&s)[4]) {
    s[0] = s[1] = s[2] = s[3] = 0.f;
    // Each scale twice.
    const Steps k0(__byte_perm(tile.ks, 0, 0x0404) >> 1), k1(__byte_perm(tile.ks, 0, 0x1414) >> 1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        const uint32_t x = ks < 2 ? tile.k.x : tile.k.y, y = ks < 2 ? tile.k.z : tile.k.w;
        const uint32_t xs = pkv::int4::swap_bytes(x), ys = pkv::int4::swap_bytes(y);
        const int i = 2 * (ks & 1);
        const uint32_t a0 = value_pair(x, xs, i, k0), a1 = value_pair(y, ys, i, k1);
        const uint32_t a2 = value_pair(x, xs, i + 1, k0), a3 = value_pair(y, ys, i + 1, k1);
        mma(s, a0, a1, a2, a3, q.high[2 * ks], q.high[2 * ks + 1]);
        if (R != Kind::kPlain) mma(s, a0, a1, a2, a3, q.low[2 * ks], q.low[2 * ks + 1]);
    }
}

// Adds the weights w of a block's tokens (rows g and g + 8 of heads 2 t, 2 t + 1) times its V.
__device__ __forceinline__ void add_values(const Tile &tile, const float (&w)[4], Sums &sums) {
    // hi: the first 11 bits, cut off by the integer pipe (the FP16 and FP32 ones are the busy ones);
    // lo: the rest.
    float hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hi[j] = __uint_as_float(__float_as_uint(w[j]) & 0xffffe000u);
        lo[j] = w[j] - hi[j];
    }
    const uint32_t p0 = pkv::movmatrix_trans(pack(__floats2half2_rn(hi[0], hi[1])));
    const uint32_t p1 = pkv::movmatrix_trans(pack(__floats2half2_rn(hi[2], hi[3])));
    const uint32_t r0 = pkv::movmatrix_trans(pack(__floats2half2_rn(lo[0], lo[1])));
    const uint32_t r1 = pkv::movmatrix_trans(pack(__floats2half2_rn(lo[2], lo[3])));
    // Tokens 4 t, 4 t + 2 in the first pair, 4 t + 1, 4 t + 3 in the second.
    const Steps v0((tile.vs & 0x00ff00ffu) << 7), v1((tile.vs & 0xff00ff00u) >> 1);
    const uint4 &v = tile.v;
    uint32_t even[4], odd[4];  // a pair's low halves, straight and swapped, and its high ones
    even[0] = __byte_perm(v.x, v.z, 0x5410), even[1] = __byte_perm(v.x, v.z, 0x4501);
    even[2] = __byte_perm(v.x, v.z, 0x7632), even[3] = __byte_perm(v.x, v.z, 0x6723);
    odd[0] = __byte_perm(v.y, v.w, 0x5410), odd[1] = __byte_perm(v.y, v.w, 0x4501);
    odd[2] = __byte_perm(v.y, v.w, 0x7632), odd[3] = __byte_perm(v.y, v.w, 0x6723);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
        const uint32_t a0 = value_pair(even[0], even[1], mt, v0), a1 = value_pair(even[2], even[3], mt, v0);
        const uint32_t a2 = value_pair(odd[0], odd[1], mt, v1), a3 = value_pair(odd[2], odd[3], mt, v1);
        mma(sums.o[mt], a0, a1, a2, a3, p0, p1);
        mma(sums.o[mt], a0, a1, a2, a3, r0, r1);
    }
}

// COUNT blocks, of which `valid` tokens count (MASKED; else all).
template <Kind R, int COUNT, bool MASKED>
__device__ __forceinline__ void attend(Tile (&tile)[COUNT], int valid, const Query &q, Sums &sums, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float s[COUNT][4], x[COUNT][4];
#pragma unroll
    for (int b = 0; b < COUNT; ++b) {
        score<R>(tile[b], q, s[b]);
        if constexpr (MASKED) {
            const int here = valid - b * kSlots;
            if (2 * g >= here) s[b][0] = s[b][1] = -INFINITY;
            if (2 * g + 1 >= here) s[b][2] = s[b][3] = -INFINITY;
            const int keep = min(max(here - 4 * t, 0), 4);  // V of masked tokens: weight 0 times NaN is NaN
            if (keep < 4) tile[b].vs &= (1u << (8 * keep)) - 1u;
        }
    }
    float most = -INFINITY;
#pragma unroll
    for (int b = 0; b < COUNT; ++b) {
        sums.exponents(s[b], q, x[b]);
        most = pkv::fmax3(pkv::fmax3(most, x[b][0], x[b][1]), x[b][2], x[b][3]);
    }
    if (__any_sync(0xffffffffu, most > kMostWeight)) {
        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
        for (int b = 0; b < COUNT; ++b) {
            top0 = fmaxf(top0, fmaxf(__fmul_rn(s[b][0], q.factor0), __fmul_rn(s[b][2], q.factor0)));
            top1 = fmaxf(top1, fmaxf(__fmul_rn(s[b][1], q.factor1), __fmul_rn(s[b][3], q.factor1)));
        }
        sums.raise(top0, top1);
#pragma unroll
        for (int b = 0; b < COUNT; ++b) sums.exponents(s[b], q, x[b]);
    }
#pragma unroll
    for (int b = 0; b < COUNT; ++b) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pkv::exp2_approx(x[b][j]);
        sums.l = pkv::add_f32x2(sums.l, pkv::add_f32x2(pkv::f32x2(w[0], w[1]), pkv::f32x2(w[2], w[3])));
        add_values(tile[b], w, sums);
    }
}

// One piece of the list.  Three CTAs an SM (four hold too few registers, and spill) and a ring of
// two stages of four blocks (three stages, stages of one block: no faster); two blocks a step give
// each warp two chains of MMAs (one and four are slower).
template <Kind R>
__global__ void __launch_bounds__(kThreads, 3) int4_decode_kernel(const __grid_constant__ ArgsOf<R> a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            pkv::mbar_init(pkv::smem_addr(&full[s]), 1);
            pkv::mbar_init(pkv::smem_addr(&empty[s]), kWarps);
        }
        pkv::fence_barrier_init();
    }
    __syncthreads();
    pkv::pdl_wait();
    pkv::pdl_launch_dependents();

    // The piece and the row that it begins in.
    const int piece = blockIdx.x;
    int begin, end, row;
    int pieces;
    if (a.batch <= kWeighedRows) {
        const RowScan scan(a, lane);
        const Cut cut(a, scan.count, scan.short_rows);
        pieces = cut.total > 0 ? cut.pieces : 0;
        if (cut.by_row) {
            scan.row_at(piece, cut.total, lane, begin, end, row);
        } else {
            int other;
            begin = scan.block_at(cut.begins(min(piece, cut.pieces)), cut.total, lane, row);
            end = scan.block_at(cut.begins(min(piece + 1, cut.pieces)), cut.total, lane, other);
        }
    } else {
        // Of 32 samples of prefix, `step` rows apart, the first past `begin`, cut finer until the
        // samples are rows.
        int step = (a.batch + 31) / 32;
        int sample = lane * step < a.batch ? a.prefix_at(min((lane + 1) * step, a.batch)) : INT32_MAX;
        const Cut cut(a, 0, false);
        pieces = cut.total > 0 ? cut.pieces : 0;
        begin = static_cast<int>(cut.begins(min(piece, cut.pieces))), end = static_cast<int>(cut.begins(min(piece + 1, cut.pieces)));
        row = 0;
        while (true) {
            const unsigned past = __ballot_sync(0xffffffffu, sample > begin);
            row += (past != 0 ? __ffs(past) - 1 : 31) * step;
            if (step == 1) {
                // In a list that is out of order the last samples may all lie before `begin`: no row
                // is taken that does not end past it.
                if (past == 0) row = INT32_MAX;
                break;
            }
            step = (step + 31) / 32;
            sample = row + lane * step < a.batch ? a.prefix_at(min(row + (lane + 1) * step, a.batch)) : INT32_MAX;
        }
    }
    // Rows without blocks: zeros, a warp looking at 32 rows.  (The merge looks at the rows' order
    // too, where there is one.)
    for (int b = (blockIdx.x * (kWarps + 1) + warp) * 32; (a.clear || a.part_o == nullptr) && b < a.batch; b += a.grid * kThreads) {
        const int r = b + lane;
        const int first = r < a.batch ? a.prefix_at(r) : 0, last = r < a.batch ? a.prefix_at(r + 1) : 1;
        if (r < a.batch && out_of_order(r, first, last)) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        for (unsigned none = __ballot_sync(0xffffffffu, last <= first); a.clear && none != 0; none &= none - 1) {
            uint4 *const out = reinterpret_cast<uint4 *>(a.out + (b + __ffs(none) - 1) * a.out_stride);
            for (int i = lane; i < kQueryHeads * kDim / 8; i += 32) out[i] = make_uint4(0, 0, 0, 0);
        }
    }
    if (piece >= pieces || begin >= end) return;
    if (row >= a.batch) {  // prefix does not grow from row to row
        if (threadIdx.x == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        return;
    }
    if (warp == kProducer) {
        fill_ring<R>(a, begin, end, row, lane, smem, full, empty);
        return;
    }
    Rows rows = load_rows(a, row, lane);

    const Places places(pkv::smem_addr(smem) + warp * pkv::int4::kHeadBytes, lane);
    uint8_t *const fresh = smem + kFreshAt + warp * kFreshBytes;
    int consumed = 0;
    bool failed = false;
    int i = begin;
    while (i < end) {
        if (row >= a.batch) {  // prefix does not grow from row to row
            if (threadIdx.x == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
            break;
        }
        const int row_first = __shfl_sync(0xffffffffu, rows.first, row - rows.base);
        const int row_last = __shfl_sync(0xffffffffu, rows.last, row - rows.base);
        const int length = __shfl_sync(0xffffffffu, rows.length, row - rows.base);
        const int seg_end = min(end, row_last);
        if (R == Kind::kFresh && row_last <= end) write_new(a, row, length, a.flat[row_last - 1], warp, lane, fresh);
        Query q;
        q.load<R>(a, row, length, warp, lane);
        int next = row;
        if (row_last < end) {  // the next row's queries are brought near while this one streams
            next = advance_row(a, rows, row + 1, row_last, lane);
            if (next < a.batch) prefetch_query<R>(a, next, warp, lane);
        }
        Sums sums;
        sums.clear();
        // The row's tokens from block i on.  (Behind its length a row may list any number of blocks: times
        // 16 they may pass 32 bits.)
        const int before = i - row_first;
        int left = before > (length >> 4) ? 0 : length - before * kSlots;
        while (i < seg_end) {
            const int n = min(kChunk, seg_end - i);
            const int stage = consumed % kStages;
            failed = !wait_bounded(pkv::smem_addr(&full[stage]), (consumed / kStages) & 1);
            failed = __any_sync(0xffffffffu, failed);
            if (failed) break;
            if (R == Kind::kFresh && i + n == row_last) {
                put_fresh(fresh, smem + stage * kStageBytes + (n - 1) * pkv::int4::kBlockBytes + warp * pkv::int4::kHeadBytes,
                          (length - 1) & (kSlots - 1), lane);
            }
            const int tokens = min(left, n * kSlots);  // valid ones of the chunk
            left -= tokens;
            const Places here = places.at(stage * kStageBytes);
            const auto release = [&] {
                // Every lane has read the stage (the fence orders the reads before the copies, the
                // warp barrier the lanes): it may be filled again.
                pkv::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) pkv::mbar_arrive(pkv::smem_addr(&empty[stage]));
            };
            if (tokens == kChunk * kSlots) {
                Tile tile[2];
                tile[0].load<0>(here);
                tile[1].load<1>(here);
                attend<R, 2, false>(tile, 0, q, sums, lane);
                tile[0].load<2>(here);
                tile[1].load<3>(here);
                release();
                attend<R, 2, false>(tile, 0, q, sums, lane);
            } else {
#pragma unroll 1
                for (int b = 0; b < n; ++b) {
                    Tile tile[1];
                    tile[0].load<0>(here.at(b * pkv::int4::kBlockBytes));
                    if (b + 1 == n) release();
                    attend<R, 1, true>(tile, tokens - b * kSlots, q, sums, lane);
                }
            }
            i += n;
            ++consumed;
        }
        if (failed) break;

        const float2 l = pkv::unpack_f32x2(sums.l);
        const float l0 = sum8(l.x), l1 = sum8(l.y);
        const auto &o = sums.o;
        const int head0 = warp * kHeadGroup + 2 * t;
        if (row_first >= begin && row_last <= end) {
            // Normalise and round; a row whose every token is masked is zeros.
            const float n0 = l0 * kValueFactor, n1 = l1 * kValueFactor;
            __half *dst = a.out + row * a.out_stride + head0 * kDim + 8 * g;
            uint32_t x[4], y[4];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                x[mt] = l0 == 0.f ? 0u : pack(__floats2half2_rn(__fdiv_rn(o[mt][0], n0), __fdiv_rn(o[mt][2], n0)));
                y[mt] = l1 == 0.f ? 0u : pack(__floats2half2_rn(__fdiv_rn(o[mt][1], n1), __fdiv_rn(o[mt][3], n1)));
            }
            *reinterpret_cast<uint4 *>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4 *>(dst + kDim) = make_uint4(y[0], y[1], y[2], y[3]);
        } else if (a.part_o == nullptr) {  // begins before the list or ends behind it
            if (lane == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        } else {
            const int64_t index = static_cast<int64_t>(row) + blockIdx.x;
            float *po = a.part_o + index * kQueryHeads * kDim + head0 * kDim + 8 * g;
            constexpr float kUndo = 1.f / kValueFactor;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 *dst = reinterpret_cast<float4 *>(po + h * kDim);
                dst[0] = make_float4(o[0][h] * kUndo, o[0][2 + h] * kUndo, o[1][h] * kUndo, o[1][2 + h] * kUndo);
                dst[1] = make_float4(o[2][h] * kUndo, o[2][2 + h] * kUndo, o[3][h] * kUndo, o[3][2 + h] * kUndo);
            }
            if (g == 0) {
                *reinterpret_cast<float4 *>(a.part_ml + index * kQueryHeads * 2 + head0 * 2) =
                    make_float4(sums.m0, l0, sums.m1, l1);
            }
        }
        row = next;
    }
    if (failed && lane == 0) atomicOr(a.error_flag, PKV_DEVICE_WAIT_TIMEOUT);
}

// Merge of the rows that several pieces hold: H half warps a (row, head), whose sixteen lanes
// hold its 64 dims, each with every H-th piece, four or eight read at a time; then the halves of a
// warp are joined, and the warps' results in order.  Bound by the latency of a launch and of two
// rounds of loads, about 2.5 us (its partials, 9 MB for 256 rows, come from L2).
template <int H>
constexpr int kMergeThreads = 16 * (H < 16 ? 16 : H);

__device__ __forceinline__ void join_halves(Merge &m) {
    const float4 v = make_float4(__shfl_down_sync(0xffffffffu, m.A[0], 16), __shfl_down_sync(0xffffffffu, m.A[1], 16),
                                 __shfl_down_sync(0xffffffffu, m.A[2], 16), __shfl_down_sync(0xffffffffu, m.A[3], 16));
    const float top = __shfl_down_sync(0xffffffffu, m.M, 16), sum = __shfl_down_sync(0xffffffffu, m.L, 16);
    m.add(top, sum, v);  // of use in the lower half
}

template <int H, Kind R>
__global__ void __launch_bounds__(kMergeThreads<H>) int4_merge_kernel(const __grid_constant__ ArgsOf<R> a) {
    __shared__ float part[H > 2 ? kMergeThreads<H> / 32 : 1][16][6];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = threadIdx.x >> 4;
    const int at = blockIdx.x * (kMergeThreads<H> / 16 / H) + half / H;
    const int row = at / kQueryHeads, head = at % kQueryHeads;
    const int dim = 4 * (lane & 15);
    pkv::pdl_launch_dependents();
    // The tables are older than the split kernel: it lets this one start only after
    // its own wait for what came before.
    int first = 0, last = 0;
    const int row_at = min(row, a.batch - 1);
    const int first_block = a.prefix_at(row_at), last_block = a.prefix_at(row_at + 1) - 1;
    int rank = 0, rows_with_blocks = 0;
    bool short_rows = false;
    if (a.batch <= kWeighedRows) {
        const RowScan scan(a, lane);
        rank = scan.rank(row_at);
        rows_with_blocks = scan.count;
        short_rows = scan.short_rows;
    }
    const Cut cut(a, rows_with_blocks, short_rows);
    if (row < a.batch) {
        if (lane == 0 && out_of_order(row, first_block, last_block + 1)) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        if (last_block >= first_block && first_block >= 0 && last_block < cut.total) {
            first = cut.piece_of(first_block, rank);
            last = min(cut.piece_of(last_block, rank), cut.pieces - 1);
        }
    }
    pkv::pdl_wait();
    if (H <= 2 && __all_sync(0xffffffffu, first >= last)) return;
    Merge merged{kLowest, 0.f, {0.f, 0.f, 0.f, 0.f}};
    constexpr int kBatch = H > 8 ? 8 : 4, kStep = H;
    for (int c0 = first + half % H; c0 <= last && first < last; c0 += kBatch * kStep) {
        float2 ml[kBatch];
        float4 v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int c = c0 + j * kStep;
            if (c <= last) {
                const int64_t index = (static_cast<int64_t>(row) + c) * kQueryHeads + head;
                ml[j] = *reinterpret_cast<const float2 *>(a.part_ml + index * 2);
                v[j] = *reinterpret_cast<const float4 *>(a.part_o + index * kDim + dim);
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (c0 + j * kStep <= last) merged.add(ml[j].x, ml[j].y, v[j]);
        }
    }
    if constexpr (H > 1) {
        __syncwarp();
        join_halves(merged);
    }
    if constexpr (H > 2) {
        constexpr int kWarpsAHead = H / 2;
        if (lane < 16) {
            float *mine = part[warp][lane];
            mine[0] = merged.M, mine[1] = merged.L;
            mine[2] = merged.A[0], mine[3] = merged.A[1], mine[4] = merged.A[2], mine[5] = merged.A[3];
        }
        __syncthreads();
        if (warp % kWarpsAHead != 0 || first >= last) return;
        merged = Merge{kLowest, 0.f, {0.f, 0.f, 0.f, 0.f}};
        for (int other = lane >> 4; other < kWarpsAHead; other += 2) {
            const float *p = part[warp + other][lane & 15];
            merged.add(p[0], p[1], make_float4(p[2], p[3], p[4], p[5]));
        }
        __syncwarp();
        join_halves(merged);
    }
    if (first >= last || (H > 1 && lane >= 16)) return;
#pragma unroll
    for (int d = 0; d < 4; ++d) merged.A[d] = merged.L == 0.f ? 0.f : __fdiv_rn(merged.A[d], merged.L);
    const __half2 low = __floats2half2_rn(merged.A[0], merged.A[1]), high = __floats2half2_rn(merged.A[2], merged.A[3]);
    *reinterpret_cast<uint2 *>(a.out + row * a.out_stride + head * kDim + dim) = make_uint2(pack(low), pack(high));
}

template <int H, Kind R>
cudaError_t launch_merge(const ArgsOf<R> &a, cudaStream_t stream) {
    constexpr int kHeadsPerCta = kMergeThreads<H> / 16 / H;
    const int64_t heads = static_cast<int64_t>(a.batch) * kQueryHeads;
    return pkv::launch_pdl(int4_merge_kernel<H, R>, dim3(static_cast<unsigned>((heads + kHeadsPerCta - 1) / kHeadsPerCta)),
                           dim3(kMergeThreads<H>), stream, a);
}

// Whether rows may be split: not one piece, nor a list so short that all of its rows are, with a
// piece for each.
bool splits_rows(int64_t batch, int64_t total, int64_t grid) {
    return grid > 1 && (total > kShortRow || batch > kWeighedRows || grid < (batch < total ? batch : total));
}

int64_t workspace_of(int64_t batch, int64_t total, int64_t grid) {
    return splits_rows(batch, total, grid) ? (batch + grid) * kPartial * 4 : 0;
}

struct DeviceInfo {
    int sms = 0;
    int ctas_per_sm = 0;
};

template <Kind R>
cudaError_t prepare_kernel(int *ctas_per_sm) {
    const auto kernel = int4_decode_kernel<R>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
    int ctas = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, kThreads, kSmem);
    if (ctas < *ctas_per_sm) *ctas_per_sm = ctas;
    return e;
}

// The merge keeps the split kernel's partition of L1 and shared memory.
template <Kind R>
cudaError_t prepare_merges() {
    cudaError_t e = cudaSuccess;
    for (const auto merge : {int4_merge_kernel<1, R>, int4_merge_kernel<2, R>, int4_merge_kernel<4, R>, int4_merge_kernel<8, R>,
                             int4_merge_kernel<32, R>}) {
        if (e == cudaSuccess) {
            e = cudaFuncSetAttribute(merge, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        }
    }
    return e;
}

constexpr int kMaxDevices = 64;

// SMs and resident CTAs of `device`, found out at its first use.
int device_info(int device, DeviceInfo *info) {
    static std::atomic<int> sms[kMaxDevices] = {}, ctas[kMaxDevices] = {};
    const bool known = device >= 0 && device < kMaxDevices;
    if (known && ctas[device].load(std::memory_order_acquire) > 0) {
        info->sms = sms[device].load(std::memory_order_relaxed);
        info->ctas_per_sm = ctas[device].load(std::memory_order_relaxed);
        return PKV_OK;
    }
    int previous = 0, least = 1 << 20;
    cudaError_t e = cudaGetDevice(&previous);
    if (e == cudaSuccess) e = cudaSetDevice(device);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 decode: ") + cudaGetErrorString(e));
    e = cudaDeviceGetAttribute(&info->sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = prepare_kernel<Kind::kPlain>(&least);
    if (e == cudaSuccess) e = prepare_kernel<Kind::kFresh>(&least);
    if (e == cudaSuccess) e = prepare_kernel<Kind::kChunk>(&least);
    if (e == cudaSuccess) e = prepare_merges<Kind::kPlain>();
    if (e == cudaSuccess) e = prepare_merges<Kind::kChunk>();
    cudaSetDevice(previous);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 decode: ") + cudaGetErrorString(e));
    info->ctas_per_sm = least < 1 ? 1 : least;
    if (known) {
        sms[device].store(info->sms, std::memory_order_relaxed);
        ctas[device].store(info->ctas_per_sm, std::memory_order_release);
    }
    return PKV_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <Kind R>
cudaError_t launch_split(const ArgsOf<R> &a, cudaStream_t stream) {
    return pkv::launch_pdl_smem(int4_decode_kernel<R>, dim3(a.grid), dim3(kThreads), kSmem, stream, a);
}

template <Kind R>
cudaError_t merge(const ArgsOf<R> &a, const DeviceInfo &info, cudaStream_t stream) {
    // Half warps a head by the pieces that a row has when the GPU is full, so that one round of
    // loads or two are enough; by nothing else, for results must not depend on the room of a
    // captured launch.  (Whole calls: 100 rows, 5 pieces each, 18.0 us with 2 and 19.9 with 4;
    // 64 rows, 7 each, 26.1 and 25.8; 7 rows, 64 each, 6.7 with 8 and 7.8 with 16; 2 rows, 222
    // each, 26.1 with 16 and 25.1 with 32.)
    const int pieces = info.sms * info.ctas_per_sm / a.batch + 1;
    return pieces <= 4 ? launch_merge<1, R>(a, stream)
        : pieces <= 6 ? launch_merge<2, R>(a, stream)
        : pieces <= 16 ? launch_merge<4, R>(a, stream)
        : pieces <= 96 ? launch_merge<8, R>(a, stream)
                       : launch_merge<32, R>(a, stream);
}

// Checks and launches; `a` holds everything but the partials' addresses.
int decode(Args a, void *workspace, int64_t workspace_bytes, cudaStream_t stream) {
    const int rc = pkv::int4::check_cache(a.cache.storage, a.cache.layers, a.cache.num_blocks, a.layer, 1);
    if (rc) return rc;
    const void *const query = a.query32 != nullptr ? static_cast<const void *>(a.query32) : a.query;
    if (query == nullptr || (a.flat == nullptr && a.capacity > 0) || a.out == nullptr || a.error_flag == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: null pointer argument");
    }
    if (a.batch < 1 || a.batch > pkv::int4::kMostRows || a.capacity < 0 || a.capacity > pkv::int4::kMostEntries ||
        a.grid < 1 || a.grid > kMostGrid) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: batch, block count or grid out of range");
    }
    if (!aligned16(query) || !aligned16(a.out) || a.query_stride % 8 || a.out_stride % 8 ||
        a.query_stride < kQueryHeads * kDim || a.out_stride < kQueryHeads * kDim) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: rows must be 16-byte aligned, 2048 or more values apart in multiples of 8");
    }
    const int64_t needed = workspace_of(a.batch, a.capacity, a.grid);
    if (needed > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < needed)) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: the workspace is too small (see pkv_int4_decode_plan)");
    }
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
    DeviceInfo info;
    if (const int failed = device_info(device, &info)) return failed;
    if (needed > 0) {
        a.part_o = static_cast<float *>(workspace);
        a.part_ml = a.part_o + (static_cast<int64_t>(a.batch) + a.grid) * kQueryHeads * kDim;
    }
    e = a.key != nullptr      ? launch_split(ArgsOf<Kind::kFresh>(a), stream)
        : a.prefix != nullptr ? launch_split(ArgsOf<Kind::kPlain>(a), stream)
                              : launch_split(ArgsOf<Kind::kChunk>(a), stream);
    if (e == cudaSuccess && needed > 0) {
        e = a.prefix != nullptr ? merge(ArgsOf<Kind::kPlain>(a), info, stream) : merge(ArgsOf<Kind::kChunk>(a), info, stream);
    }
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 decode launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

Args args_of(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer, const void *query,
             int64_t query_stride, const int32_t *lengths, const int32_t *prefix, const int32_t *flat, int32_t batch,
             int32_t total_blocks, int32_t grid, void *out, int64_t out_stride, int32_t *error_flag) {
    Args a = {};
    a.cache = pkv::int4::cache_of(storage, layers, num_blocks);
    a.layer = layer;
    a.query = static_cast<const __half *>(query);
    a.query_stride = query_stride;
    a.lengths = lengths;
    a.prefix = prefix;
    a.flat = flat;
    a.batch = batch;
    a.capacity = total_blocks;
    a.grid = grid;
    a.clear = 1;
    a.out = static_cast<__half *>(out);
    a.out_stride = out_stride;
    a.error_flag = error_flag;
    return a;
}

}  // namespace

namespace pkv::int4 {

int rows_workspace(int device, int start, int tokens, int64_t *bytes) {
    int32_t grid = 0;
    return pkv_int4_decode_plan(device, tokens, blocks_before(start, tokens), &grid, bytes);
}

int attend_rows(const Cache &cache, int32_t layer, const void *query, bool query_fp32, int64_t query_stride,
                const int32_t *blocks, int32_t start, int32_t tokens, void *out, int64_t out_stride, void *workspace,
                int64_t workspace_bytes, int32_t *error_flag, cudaStream_t stream) {
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return fail(PKV_CUDA_ERROR, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
    const int total = blocks_before(start, tokens);
    int32_t grid = 0;
    int64_t needed = 0;
    if (const int rc = pkv_int4_decode_plan(device, tokens, total, &grid, &needed)) return rc;
    Args a = args_of(cache.storage, cache.layers, cache.num_blocks, layer, query_fp32 ? nullptr : query, query_stride, nullptr,
                     nullptr, blocks, tokens, total, grid, out, out_stride, error_flag);
    if (query_fp32) a.query32 = static_cast<const float *>(query);
    a.start = start;
    return decode(a, workspace, workspace_bytes, stream);
}

}  // namespace pkv::int4

extern "C" int pkv_int4_decode_plan(int32_t device, int32_t batch, int32_t total_blocks, int32_t *out_grid,
                                    int64_t *out_workspace_bytes) {
    pkv::clear_error();
    if (out_grid == nullptr || out_workspace_bytes == nullptr || batch < 1 || total_blocks < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode plan: needs a nonempty batch");
    }
    if (batch > pkv::int4::kMostRows || total_blocks > pkv::int4::kMostEntries) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode plan: batch or block count out of range");
    }
    DeviceInfo info;
    const int rc = device_info(device, &info);
    if (rc) return rc;
    // At most one CTA per resident slot.  (A list of short rows needs no merge: one of 5 blocks takes
    // 4.7 us, in two pieces 5.8.)
    const int slots = info.sms * info.ctas_per_sm;
    const int grid = total_blocks > kShortRow || batch > kWeighedRows
        ? pieces_of(total_blocks, batch <= kWeighedRows ? batch : total_blocks, slots)
        : std::max(1, std::min({batch, total_blocks, slots}));
    *out_grid = grid;
    *out_workspace_bytes = workspace_of(batch, total_blocks, grid);
    return PKV_OK;
}

extern "C" int pkv_int4_decode_attention(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer,
                                         const void *query, int64_t query_stride, const int32_t *lengths,
                                         const int32_t *prefix, const int32_t *flat, int32_t batch,
                                         int32_t total_blocks, int32_t grid, void *out, int64_t out_stride,
                                         void *workspace, int64_t workspace_bytes, int32_t *error_flag, void *stream) {
    pkv::clear_error();
    if (lengths == nullptr || prefix == nullptr) return pkv::fail(PKV_VALUE_ERROR, "int4 decode: null pointer argument");
    return decode(args_of(storage, layers, num_blocks, layer, query, query_stride, lengths, prefix, flat, batch,
                          total_blocks, grid, out, out_stride, error_flag),
                  workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int pkv_int4_decode_layer(void *storage, int32_t layers, int32_t num_blocks, int32_t layer, const void *query,
                                     int64_t query_stride, const void *key, const void *value, int64_t kv_stride,
                                     const void *rope_table, const void *query_norm, const void *key_norm, double eps,
                                     const int32_t *lengths, const int32_t *prefix, const int32_t *flat, int32_t batch,
                                     int32_t total_blocks, int32_t grid, int32_t clear, void *out, int64_t out_stride,
                                     void *workspace, int64_t workspace_bytes, int32_t *error_flag, void *stream) {
    pkv::clear_error();
    if (lengths == nullptr || prefix == nullptr) return pkv::fail(PKV_VALUE_ERROR, "int4 decode: null pointer argument");
    if (key == nullptr || value == nullptr || rope_table == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode layer: key, value and rope_table are required");
    }
    if (!aligned16(key) || !aligned16(value) || kv_stride % 8 || !aligned16(rope_table)) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode layer: new K/V rows must be 16-byte aligned with strides in multiples of 8");
    }
    if ((query_norm != nullptr) != (key_norm != nullptr) || !aligned16(query_norm) || !aligned16(key_norm)) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode layer: the norms go together, 16-byte aligned");
    }
    Args a = args_of(storage, layers, num_blocks, layer, query, query_stride, lengths, prefix, flat, batch, total_blocks,
                     grid, out, out_stride, error_flag);
    a.key = static_cast<const __half *>(key);
    a.value = static_cast<const __half *>(value);
    a.kv_stride = kv_stride;
    a.rope = static_cast<const __half *>(rope_table);
    const int64_t at = static_cast<int64_t>(layer) * kDim;
    a.query_norm = query_norm != nullptr ? static_cast<const __half *>(query_norm) + at : nullptr;
    a.key_norm = key_norm != nullptr ? static_cast<const __half *>(key_norm) + at : nullptr;
    a.eps = eps;
    a.clear = clear;
    return decode(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
