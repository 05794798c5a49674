// Batched one-token attention over the 4-bit KV cache (numbers and layout: int4.cuh):
//   out[b, h] = sum_t softmax_t(q[b, h] . K[t, h / 8] / 8) V[t, h / 8]
// over the lengths[b] tokens that row b's block table lists; for a decode layer the row's new
// token is written first, its K and the row's queries normed (where asked for) and rotated here.
//
// Work split: the batch's block tables form one flat list, CTA g streams piece g of it, warp w
// serves KV head w and its eight query heads.  A row that one piece holds is written directly;
// the others leave (m, l, O) partials at index row + piece (unique: along the pieces the pairs
// form a monotone staircase) that a second kernel merges in piece order.
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
// Weights and the layer's queries go in as two FP16 numbers each, hi = fp16(x) and
// lo = fp16(x - hi), 2^-22 of x together (one alone shows in the output beside its own
// rounding); a query head is scaled by the power of two that brings its largest value to
// 2^14 .. 2^15 first, whatever its range.  Scores, maxima, normaliser and sums are FP32.

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
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
constexpr int kWarps = kHeads;
constexpr int kThreads = kWarps * 32;
constexpr int kLeastPiece = 4;  // blocks
constexpr float kScaleLog2 = 0.125f * 1.4426950408889634f;  // 64^-0.5 * log2(e)
constexpr float kValueFactor = 0x1p-6f;  // of the values in the MMAs
constexpr float kWeightShift = 15.0f;
constexpr float kFarScore = 0x1p20f;
constexpr float kLowest = -1e30f;  // below every finite score
constexpr int kPartial = kQueryHeads * (kDim + 2);  // floats of a partial

struct Args {
    pkv::int4::Cache cache;
    int32_t layer;
    const __half *query;
    int64_t query_stride;
    const __half *key;  // the new tokens, with rope; null for the attention alone
    const __half *value;
    int64_t kv_stride;
    const __half *rope;
    const __half *query_norm;  // of this layer, or null
    const __half *key_norm;
    double eps;
    const int32_t *lengths;
    const int32_t *prefix;
    const int32_t *flat;
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

// Piece g covers blocks [g * total / pieces, (g + 1) * total / pieces).
__device__ __forceinline__ int piece_begin(int g, int total, int pieces) {
    return static_cast<int>(static_cast<int64_t>(g) * total / pieces);
}

__device__ __forceinline__ int piece_of(int block, int total, int pieces) {
    return static_cast<int>(((static_cast<int64_t>(block) + 1) * pieces - 1) / total);
}

// Pieces of a list of `total` blocks: at most one per CTA and per kLeastPiece blocks, so
// none is empty.  (A captured launch has a CTA for every resident slot.)
__host__ __device__ __forceinline__ int pieces_of(int total, int grid) {
    const int most = (total + kLeastPiece - 1) / kLeastPiece;
    return most < 1 ? 1 : most < grid ? most : grid;
}

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

    template <bool NEW>
    __device__ __forceinline__ void load(const Args &a, int row, int length, int warp, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const __half *src = a.query + row * a.query_stride + (warp * kHeadGroup + g) * kDim;
        if constexpr (!NEW) {
            const uint4 *from = reinterpret_cast<const uint4 *>(src + 16 * t);
            const uint4 x = from[0], y = from[1];
            high[0] = x.x, high[1] = x.y, high[2] = x.z, high[3] = x.w;
            high[4] = y.x, high[5] = y.y, high[6] = y.z, high[7] = y.w;
            factor0 = factor1 = kScaleLog2 / kValueFactor;
            return;
        }
        float q[16], other[16], cos[16], sin[16];
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
        float largest = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            q[i] = q[i] * cos[i] + (t < 2 ? -other[i] : other[i]) * sin[i];
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

// The new token of row `row` into its slot of the row's last block: K by lanes 0 .. 3 of the
// head's warp, V by lanes 4 .. 7.
__device__ __forceinline__ void write_new(const Args &a, int row, int length, int last_block, int warp, int lane) {
    const int t = lane & 3;
    const int block = a.flat[last_block];
    const bool ok = block >= 0 && block < a.cache.num_blocks && length >= 1 && length <= PKV_CONTEXT_LIMIT;
    if (!ok) {
        if (warp == 0 && lane == 0) {
            atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
            if (length < 1 || length > PKV_CONTEXT_LIMIT) atomicOr(a.error_flag, PKV_DEVICE_BAD_POSITION);
        }
        return;
    }
    const int64_t from = row * a.kv_stride + warp * kDim;
    uint8_t *const to = pkv::int4::block_at(a.cache, a.layer, block) + warp * pkv::int4::kHeadBytes;
    const int slot = (length - 1) % kSlots;
    float v[16];
    uint32_t words[2], scale;
    pkv::int4::key_group(a.key + from, t, lane < 4, a.key_norm, a.eps, a.rope, length - 1, v);
    if (lane >= 4 && lane < 8) pkv::int4::load16(a.value + from + 16 * t, v);
    if (lane < 8) {
        pkv::int4::encode_group(v, words, scale);
        if (lane < 4) pkv::int4::store_key(to, t, slot, words, scale);
        else pkv::int4::store_value(to, t, slot, words, scale);
    }
}

template <bool NEW>
__global__ void __launch_bounds__(kThreads) int4_decode_kernel(const __grid_constant__ Args a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    pkv::pdl_wait();
    pkv::pdl_launch_dependents();
    const int total = total_blocks(a);
    const int pieces = pieces_of(total, a.grid);
    // Rows without blocks: zeros.  (The merge looks at the rows' order too, where there is one.)
    for (int b = blockIdx.x * kThreads + threadIdx.x; (a.clear || a.grid == 1) && b < a.batch; b += a.grid * kThreads) {
        const int first = a.prefix[b], last = a.prefix[b + 1];
        if (out_of_order(b, first, last)) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        if (a.clear && last <= first) {
            for (int i = 0; i < kQueryHeads * kDim; ++i) a.out[b * a.out_stride + i] = __float2half_rn(0.f);
        }
    }
    if (total == 0 || static_cast<int>(blockIdx.x) >= pieces) return;
    const int begin = piece_begin(blockIdx.x, total, pieces);
    const int end = piece_begin(blockIdx.x + 1, total, pieces);
    Rows rows = load_rows(a, 0, lane);
    int row = advance_row(a, rows, 0, begin, lane);
    for (int i = begin; i < end;) {
        if (row >= a.batch) {  // prefix does not grow from row to row
            if (threadIdx.x == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
            return;
        }
        const int row_first = __shfl_sync(0xffffffffu, rows.first, row - rows.base);
        const int row_last = __shfl_sync(0xffffffffu, rows.last, row - rows.base);
        const int length = __shfl_sync(0xffffffffu, rows.length, row - rows.base);
        const int seg_end = min(end, row_last);
        if (NEW && row_last <= end) {
            write_new(a, row, length, row_last - 1, warp, lane);
            __syncwarp();
        }
        Query q;
        q.load<NEW>(a, row, length, warp, lane);

        float m0 = kLowest, m1 = kLowest, l0 = 0.f, l1 = 0.f;
        float o[4][4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
        for (; i < seg_end; ++i) {
            const int block = a.flat[i];
            const bool bad = block < 0 || block >= a.cache.num_blocks;  // reported, and read as zeros
            if (bad && threadIdx.x == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
            const uint8_t *from = pkv::int4::block_at(a.cache, a.layer, bad ? 0 : block) + warp * pkv::int4::kHeadBytes;
            const uint4 k = *reinterpret_cast<const uint4 *>(from + pkv::int4::key_words(t, 2 * g));
            const uint4 v = *reinterpret_cast<const uint4 *>(from + pkv::int4::kValueAt + lane * 16);
            uint32_t ks = *reinterpret_cast<const uint16_t *>(from + pkv::int4::scale_at(pkv::int4::kKeyScaleAt, t, 2 * g));
            uint32_t vs = *reinterpret_cast<const uint32_t *>(from + pkv::int4::scale_at(pkv::int4::kValueScaleAt, g >> 1, 4 * t));
            if (bad) ks = vs = 0;
            const int valid = min(max(length - (i - row_first) * kSlots, 0), kSlots);  // tokens of this block
            if (valid < kSlots) {  // weight 0 times NaN is NaN
                const int keep = min(max(valid - 4 * t, 0), 4);
                vs = keep == 4 ? vs : vs & ((1u << (8 * keep)) - 1u);
            }

            float s[4] = {0.f, 0.f, 0.f, 0.f};
            const Steps k0((ks & 0xffu) * 0x00800080u), k1((ks >> 8) * 0x00800080u);  // each scale twice
#pragma unroll
            for (int ks4 = 0; ks4 < 4; ++ks4) {
                const uint32_t x = ks4 < 2 ? k.x : k.y, y = ks4 < 2 ? k.z : k.w;
                const uint32_t xs = pkv::int4::swap_bytes(x), ys = pkv::int4::swap_bytes(y);
                const int i0 = 2 * (ks4 & 1);
                const uint32_t a0 = value_pair(x, xs, i0, k0), a1 = value_pair(y, ys, i0, k1);
                const uint32_t a2 = value_pair(x, xs, i0 + 1, k0), a3 = value_pair(y, ys, i0 + 1, k1);
                mma(s, a0, a1, a2, a3, q.high[2 * ks4], q.high[2 * ks4 + 1]);
                if (NEW) mma(s, a0, a1, a2, a3, q.low[2 * ks4], q.low[2 * ks4 + 1]);
            }
            s[0] *= q.factor0, s[1] *= q.factor1, s[2] *= q.factor0, s[3] *= q.factor1;
            if (2 * g >= valid) s[0] = s[1] = -INFINITY;
            if (2 * g + 1 >= valid) s[2] = s[3] = -INFINITY;
            float top0 = max8(fmaxf(s[0], s[2])), top1 = max8(fmaxf(s[1], s[3]));
            // The reference is 15 below the maximum, so that weights reach 2^15; far out,
            // where 15 would soon be lost in its rounding, the maximum itself.
            top0 = fmaxf(m0, fabsf(top0) > kFarScore ? top0 : top0 - kWeightShift);
            top1 = fmaxf(m1, fabsf(top1) > kFarScore ? top1 : top1 - kWeightShift);
            const float alpha0 = pkv::exp2_approx(m0 - top0), alpha1 = pkv::exp2_approx(m1 - top1);
            m0 = top0;
            m1 = top1;
            const float w0 = pkv::exp2_approx(s[0] - m0), w1 = pkv::exp2_approx(s[1] - m1);
            const float w2 = pkv::exp2_approx(s[2] - m0), w3 = pkv::exp2_approx(s[3] - m1);
            l0 = fmaf(l0, alpha0, w0 + w2);
            l1 = fmaf(l1, alpha1, w1 + w3);
            const __half2 h01 = __floats2half2_rn(w0, w1), h23 = __floats2half2_rn(w2, w3);
            const float2 f01 = __half22float2(h01), f23 = __half22float2(h23);
            const uint32_t p0 = pkv::movmatrix_trans(pack(h01)), p1 = pkv::movmatrix_trans(pack(h23));
            const uint32_t r0 = pkv::movmatrix_trans(pack(__floats2half2_rn(w0 - f01.x, w1 - f01.y)));
            const uint32_t r1 = pkv::movmatrix_trans(pack(__floats2half2_rn(w2 - f23.x, w3 - f23.y)));

            // Tokens 4 t, 4 t + 2 in the first pair, 4 t + 1, 4 t + 3 in the second.
            const Steps v0((vs & 0x00ff00ffu) << 7), v1((vs & 0xff00ff00u) >> 1);
            uint32_t even[4], odd[4];  // the first pair's low and high halves, straight and swapped; the second's
            even[0] = __byte_perm(v.x, v.z, 0x5410), even[1] = __byte_perm(v.x, v.z, 0x4501);
            even[2] = __byte_perm(v.x, v.z, 0x7632), even[3] = __byte_perm(v.x, v.z, 0x6723);
            odd[0] = __byte_perm(v.y, v.w, 0x5410), odd[1] = __byte_perm(v.y, v.w, 0x4501);
            odd[2] = __byte_perm(v.y, v.w, 0x7632), odd[3] = __byte_perm(v.y, v.w, 0x6723);
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                o[mt][0] *= alpha0, o[mt][1] *= alpha1, o[mt][2] *= alpha0, o[mt][3] *= alpha1;
                const uint32_t a0 = value_pair(even[0], even[1], mt, v0), a1 = value_pair(even[2], even[3], mt, v0);
                const uint32_t a2 = value_pair(odd[0], odd[1], mt, v1), a3 = value_pair(odd[2], odd[3], mt, v1);
                mma(o[mt], a0, a1, a2, a3, p0, p1);
                mma(o[mt], a0, a1, a2, a3, r0, r1);
            }
        }

        l0 = sum8(l0);
        l1 = sum8(l1);
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
        } else if (pieces == 1) {  // begins before the list or ends behind it
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
                *reinterpret_cast<float4 *>(a.part_ml + index * kQueryHeads * 2 + head0 * 2) = make_float4(m0, l0, m1, l1);
            }
        }
        if (row_last < end) row = advance_row(a, rows, row + 1, row_last, lane);
    }
}

// Merge of the rows that several pieces hold, sixteen lanes a head and four dims a lane.
// With few rows a CTA's eight warps deal out the pieces of one (row, two heads) and the first
// warp merges the warps' results in order; with many rows a warp merges a row's few pieces.
constexpr int kMergeWarps = 8;
constexpr int kMergeThreads = kMergeWarps * 32;

template <bool SPREAD>
__global__ void __launch_bounds__(kMergeThreads) int4_merge_kernel(const __grid_constant__ Args a) {
    __shared__ float part[kMergeWarps][32][6];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pair = SPREAD ? blockIdx.x : blockIdx.x * kMergeWarps + warp;
    const int row = pair / (kQueryHeads / 2);
    const int head = 2 * (pair % (kQueryHeads / 2)) + (lane >> 4);
    const int dim = 4 * (lane & 15);
    pkv::pdl_launch_dependents();
    // The tables are older than the split kernel: it lets this one start only after
    // its own wait for what came before.
    int first = 0, last = 0;
    if (row < a.batch) {
        const int first_block = a.prefix[row], last_block = a.prefix[row + 1] - 1;
        const int total = total_blocks(a);
        if (lane == 0 && out_of_order(row, first_block, last_block + 1)) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        if (last_block >= first_block && first_block >= 0 && last_block < total) {
            const int pieces = pieces_of(total, a.grid);
            first = piece_of(first_block, total, pieces);
            last = piece_of(last_block, total, pieces);
        }
    }
    pkv::pdl_wait();
    if (first == last) return;
    constexpr int kStep = SPREAD ? kMergeWarps : 1;
    Merge merged{kLowest, 0.f, {0.f, 0.f, 0.f, 0.f}};
    constexpr int kBatch = 4;
    for (int c0 = first + (SPREAD ? warp : 0); c0 <= last; c0 += kBatch * kStep) {
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
    if constexpr (SPREAD) {
        float *mine = part[warp][lane];
        mine[0] = merged.M, mine[1] = merged.L;
        mine[2] = merged.A[0], mine[3] = merged.A[1], mine[4] = merged.A[2], mine[5] = merged.A[3];
        __syncthreads();
        if (warp != 0) return;
        for (int w = 1; w < kMergeWarps; ++w) {
            const float *p = part[w][lane];
            merged.add(p[0], p[1], make_float4(p[2], p[3], p[4], p[5]));
        }
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) merged.A[d] = merged.L == 0.f ? 0.f : __fdiv_rn(merged.A[d], merged.L);
    __half2 *dst = reinterpret_cast<__half2 *>(a.out + row * a.out_stride + head * kDim + dim);
    dst[0] = __floats2half2_rn(merged.A[0], merged.A[1]);
    dst[1] = __floats2half2_rn(merged.A[2], merged.A[3]);
}

int64_t workspace_of(int64_t batch, int64_t grid) { return grid > 1 ? (batch + grid) * kPartial * 4 : 0; }

struct DeviceInfo {
    int sms = 0;
    int ctas_per_sm = 0;
};

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
    int previous = 0, plain = 0, fresh = 0;
    cudaError_t e = cudaGetDevice(&previous);
    if (e == cudaSuccess) e = cudaSetDevice(device);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 decode: ") + cudaGetErrorString(e));
    e = cudaDeviceGetAttribute(&info->sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&plain, int4_decode_kernel<false>, kThreads, 0);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fresh, int4_decode_kernel<true>, kThreads, 0);
    cudaSetDevice(previous);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("int4 decode: ") + cudaGetErrorString(e));
    const int least = plain < fresh ? plain : fresh;
    info->ctas_per_sm = least < 1 ? 1 : least;
    if (known) {
        sms[device].store(info->sms, std::memory_order_relaxed);
        ctas[device].store(info->ctas_per_sm, std::memory_order_release);
    }
    return PKV_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks and launches; `a` holds everything but the partials' addresses.
int decode(Args a, void *workspace, int64_t workspace_bytes, cudaStream_t stream) {
    const int rc = pkv::int4::check_cache(a.cache.storage, a.cache.layers, a.cache.num_blocks, a.layer, 1);
    if (rc) return rc;
    if (a.query == nullptr || a.lengths == nullptr || a.prefix == nullptr || (a.flat == nullptr && a.capacity > 0) ||
        a.out == nullptr || a.error_flag == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: null pointer argument");
    }
    if (a.batch < 1 || a.capacity < 0 || a.grid < 1) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: batch, block count or grid out of range");
    }
    if (!aligned16(a.query) || !aligned16(a.out) || a.query_stride % 8 || a.out_stride % 8 ||
        a.query_stride < kQueryHeads * kDim || a.out_stride < kQueryHeads * kDim) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode: rows must be 16-byte aligned, 2048 or more values apart in multiples of 8");
    }
    const int64_t needed = workspace_of(a.batch, a.grid);
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
    e = pkv::launch_pdl(a.key != nullptr ? int4_decode_kernel<true> : int4_decode_kernel<false>, dim3(a.grid),
                        dim3(kThreads), stream, a);
    if (e == cudaSuccess && a.grid > 1) {
        // A CTA per (row, two heads) while that is at most two waves of CTAs: beyond it rows
        // have few pieces each and a warp merges them as fast.
        const int64_t pairs = static_cast<int64_t>(a.batch) * (kQueryHeads / 2);
        const bool spread = pairs <= 16 * info.sms;
        const auto blocks = static_cast<unsigned>(spread ? pairs : (pairs + kMergeWarps - 1) / kMergeWarps);
        e = pkv::launch_pdl(spread ? int4_merge_kernel<true> : int4_merge_kernel<false>, dim3(blocks), dim3(kMergeThreads),
                            stream, a);
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

extern "C" int pkv_int4_decode_plan(int32_t device, int32_t batch, int32_t total_blocks, int32_t *out_grid,
                                    int64_t *out_workspace_bytes) {
    pkv::clear_error();
    if (out_grid == nullptr || out_workspace_bytes == nullptr || batch < 1 || total_blocks < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "int4 decode plan: needs a nonempty batch");
    }
    DeviceInfo info;
    const int rc = device_info(device, &info);
    if (rc) return rc;
    const int grid = pieces_of(total_blocks, info.sms * info.ctas_per_sm);  // at most one CTA per resident slot
    *out_grid = grid;
    *out_workspace_bytes = workspace_of(batch, grid);
    return PKV_OK;
}

extern "C" int pkv_int4_decode_attention(const void *storage, int32_t layers, int32_t num_blocks, int32_t layer,
                                         const void *query, int64_t query_stride, const int32_t *lengths,
                                         const int32_t *prefix, const int32_t *flat, int32_t batch,
                                         int32_t total_blocks, int32_t grid, void *out, int64_t out_stride,
                                         void *workspace, int64_t workspace_bytes, int32_t *error_flag, void *stream) {
    pkv::clear_error();
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
