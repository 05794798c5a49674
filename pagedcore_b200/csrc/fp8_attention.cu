// Batched one-token attention over the 8-bit KV cache (layout: fp8_cache.cuh):
//   out[b, h] = sum_t softmax_t(q[b, h] . K[t, h / 8] / 8) V[t, h / 8]
// over the lengths[b] tokens that row b's block table lists, K and V being the
// cache's codes times their block's scale.
//
// Work split, as in the FP16 kernel: the batch's block tables form one flat
// list, CTA g streams piece g of it (equal pieces), warp w serves KV head w and
// its eight query heads.  A row that one piece holds is written directly; the
// others leave (m, l, O) partials at index row + piece (unique: along the
// pieces the pairs form a monotone staircase) that a second kernel, launched
// as its programmatic dependent, merges in piece order.
//
// Data movement: a fifth warp fills a ring of stages of up to four blocks (64
// tokens) for the whole CTA: per block one bulk copy each for the K tiles and the V
// tiles of the four heads (4 KiB, contiguous) and for the two 16-byte scale rows.
// (Copies of 1 KiB by each of the four warps were four times as many; a bulk copy
// takes the SM about 13 clocks to issue, 1.4 us for the first chunk of 12 warps.)
// V blocks lie 4128 bytes apart in a stage, so the 16-byte reads below are free of
// bank conflicts.  Two stages and three CTAs an SM keep about 200 KB under way.
//
// Math: mma.sync m16n8k16 on FP16 operands made from codes in registers
// (E4M3 to FP16 is exact), FP32 sums:
//   S^T[16 tok x 8 heads]  = K[16 x 64] . Q^T[64 x 8]
//   O^T[64 dims x 8 heads] += V^T[64 x 16] . P^T[16 x 8]
// The summed indices may be taken in any order, so each lane reads 16
// consecutive codes: in the first product lane (g, t) holds dims 16 t .. +15 of
// two tokens of block g / 2, in the second all 16 tokens of block t for dims
// g + 8 i; MMA j of either covers tokens 4 j .. 4 j + 3 of the four blocks, and the
// S^T accumulator becomes the P^T operand with two 8 x 8 transposes.
//
// Scales: K's multiplies the score.  V's, 2^e of the token's block, goes into
// the exponent: the weight is w = 2^(s + e - M + 15) with M the running maximum
// of s + e, so the largest contribution, not the largest probability, sits at
// 2^15 and blocks of very different magnitude lose nothing; the normaliser adds
// w * 2^-e, in FP32.  (M is held as M - 15.  Past 2^20, where 15 would soon be lost in
// its rounding and a weight pass FP16's range, as M itself.)  The weights go into the
// MMA as two FP16 numbers, hi = fp16(w) and lo = fp16(w - hi), 2^-22 of the weight
// together (one alone is off by 2^-11, which showed in the output), and so do the
// queries of the decode layer, rotated in FP32 and halved (two components near FP16's
// largest number rotate past it); scores, maxima, normaliser and sums are FP32.  The
// second products are free: the tensor pipe was 13 % busy without them, 25 % with them.

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>
#include <string>

#include "block_list.cuh"
#include "fp8_cache.cuh"
#include "pdl.h"
#include "ptx.cuh"
#include "status.h"

namespace {

using pkv::advance_row, pkv::load_rows, pkv::max8, pkv::Merge, pkv::out_of_order, pkv::Rows, pkv::sum8, pkv::total_blocks;

constexpr int kDim = PKV_HEAD_DIM;
constexpr int kHeads = PKV_KV_HEADS;
constexpr int kQueryHeads = PKV_QUERY_HEADS;
constexpr int kGroup = kQueryHeads / kHeads;
constexpr int kSlots = PKV_BLOCK_TOKENS;
constexpr int kTile = pkv::fp8::kTileBytes;
constexpr int kWarps = kHeads;        // consumers, one per KV head
constexpr int kProducer = kWarps;     // the warp that fills the ring
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kChunk = 4;             // blocks per stage
constexpr int kStages = 2;
constexpr int kBlockBytes = kHeads * kTile;
constexpr int kValuePitch = kBlockBytes + 32;
constexpr int kValueAt = kChunk * kBlockBytes;
constexpr int kScaleAt = kValueAt + kChunk * kValuePitch;  // K then V scale rows, 16 bytes a block
constexpr int kStageBytes = kScaleAt + 2 * kChunk * 16;
constexpr int kBlockTraffic = 2 * kBlockBytes + 32;
constexpr int kLowAt = kStages * kStageBytes;  // SPLIT_Q: the low halves of the row's queries, 32 bytes a lane
constexpr int kSmem = kLowAt + kWarps * 32 * 32;
constexpr uint32_t kWaitPolls = 1u << 24;
constexpr float kScaleLog2 = 0.125f * 1.4426950408889634f;  // 64^-0.5 * log2(e)
constexpr float kWeightShift = 15.0f;
constexpr float kFarScore = 0x1p20f;
constexpr float kLowest = -1e30f;  // below every finite score
constexpr int kPartial = kQueryHeads * (kDim + 2);  // floats of a partial

struct Args {
    pkv::fp8::Cache cache;
    int32_t layer;
    const __half *query;
    const __half *query_low;  // SPLIT_Q: query holds half of each value, this what FP16 left of it
    int64_t query_stride;
    const int32_t *lengths;
    const int32_t *prefix;
    const int32_t *flat;
    int32_t batch;
    int32_t capacity;  // of flat; the batch's blocks are prefix[batch]
    int32_t grid;
    int32_t clear;     // rows without blocks give zeros (else they are left alone)
    int32_t early;     // the kernel before this one writes, of what this one reads, only the queries and the rows' last blocks
    __half *out;
    int64_t out_stride;
    float *part_o;   // [batch + grid][32][64]
    float *part_ml;  // [batch + grid][32][2]
    int32_t *error_flag;

    __device__ __forceinline__ int prefix_at(int row) const { return prefix[row]; }
    __device__ __forceinline__ int length_at(int row) const { return lengths[row]; }
};

// Piece g covers blocks [g * total / grid, (g + 1) * total / grid).
__host__ __device__ __forceinline__ int piece_begin(int g, int total, int grid) {
    return static_cast<int>(static_cast<int64_t>(g) * total / grid);
}

__device__ __forceinline__ int piece_of(int block, int total, int grid) {
    return static_cast<int>(((static_cast<int64_t>(block) + 1) * grid - 1) / total);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar,
                                          uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy)
        : "memory");
}

// D = A(16x16, row) * B(16x8, col) + D, FP16 operands; free to move, unlike the volatile form.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word(const uint4 &v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// The low `keep` (0 .. 16) bytes of v.
__device__ __forceinline__ uint4 keep_bytes(const uint4 &v, int keep) {
    uint32_t m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = min(max(keep - 4 * i, 0), 4);
        m[i] = k == 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
    }
    return make_uint4(v.x & m[0], v.y & m[1], v.z & m[2], v.w & m[3]);
}

// Pieces of a list of `total` blocks: at most one per CTA and per chunk, so
// none is empty.  (A captured launch has a CTA for every resident slot.)
__host__ __device__ __forceinline__ int pieces_of(int total, int grid) {
    const int chunks = (total + kChunk - 1) / kChunk;
    return chunks < 1 ? 1 : chunks < grid ? chunks : grid;
}

// A lane's 16 query dims of a head: the high halves to registers, the low ones to its
// own 32 bytes of shared memory at `low`.
template <bool SPLIT_Q>
__device__ __forceinline__ void load_query(const Args &a, int row, int head, int t, uint32_t (&q)[8], uint32_t low) {
    const int64_t at = row * a.query_stride + head * kDim + 16 * t;
    const uint4 *src = reinterpret_cast<const uint4 *>(a.query + at);
    const uint4 x = src[0], y = src[1];
    if (SPLIT_Q) {
        const uint4 *rest = reinterpret_cast<const uint4 *>(a.query_low + at);
        const uint4 u = rest[0], v = rest[1];
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(low), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(low + 16), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
    q[0] = x.x, q[1] = x.y, q[2] = x.z, q[3] = x.w;
    q[4] = y.x, q[5] = y.y, q[6] = y.z, q[7] = y.w;
}

// Bring the same into L1 ahead of the row (registers for a second row do not fit).
template <bool SPLIT_Q>
__device__ __forceinline__ void prefetch_query(const Args &a, int row, int head, int t) {
    const int64_t at = row * a.query_stride + head * kDim + 16 * t;
    asm volatile("prefetch.global.L1 [%0];" ::"l"(a.query + at));
    if (SPLIT_Q) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.query_low + at));
}

// Read where it is used (volatile): the eight registers of a whole row do not fit beside the rest.
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}

__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity) {
    return pkv::mbar_test_wait(bar, parity) || pkv::mbar_wait_bounded(bar, parity, kWaitPolls);
}

// What a block id outside the cache reads as: codes of zero with the smallest scale, so
// that the block does not move the reference of the weights (the scale goes into it).
__device__ __align__(16) const uint8_t kZeroTiles[kBlockBytes] = {};
__device__ __align__(16) const float kLeastScales[kHeads] = {0x1p-15f, 0x1p-15f, 0x1p-15f, 0x1p-15f};

// The producer warp: copies the blocks of [begin, end) chunk by chunk, a chunk
// ending with its row.  `lo` is at most 32 rows before the piece's first; !ready:
// rows' last blocks only after the grid before this one.
__device__ __forceinline__ void fill_ring(const Args &a, int begin, int end, int lo, bool ready, int lane,
                                          uint8_t *smem, uint64_t *full, uint64_t *empty) {
    const uint64_t policy = pkv::l2_policy_evict_first();
    const uint32_t ring = pkv::smem_addr(smem);
    // The ids of the list's next 64 blocks, 32 at a time, a window ahead.
    int ids_base = begin;
    int ids = begin + lane < end ? a.flat[begin + lane] : 0;
    int ids_next = begin + 32 + lane < end ? a.flat[begin + 32 + lane] : 0;
    Rows rows = load_rows(a, lo, lane);
    int row = advance_row(a, rows, lo, begin, lane);
    int row_end = __shfl_sync(0xffffffffu, rows.last, row - rows.base);
    const int64_t layer_tile = pkv::fp8::tile_index(a.cache, a.layer, 0, 0);
    int issued = 0;
    bool ok = true;
    for (int at = begin; at < end;) {
        if (at >= row_end) {
            row = advance_row(a, rows, row + 1, at, lane);
            row_end = __shfl_sync(0xffffffffu, rows.last, row - rows.base);
        }
        if (row >= a.batch) break;  // prefix does not grow from row to row: the consumers stop here too
        const int n = min(kChunk, min(row_end, end) - at);
        if (at - ids_base >= 32) {
            ids = ids_next;
            ids_base += 32;
            const int ahead = ids_base + 32 + lane;
            ids_next = ahead < end ? a.flat[ahead] : 0;
        }
        const int j = lane & 3;
        const int offset = at - ids_base + j;
        const int near = __shfl_sync(0xffffffffu, ids, offset & 31);
        const int far = __shfl_sync(0xffffffffu, ids_next, offset & 31);
        const int block = offset < 32 ? near : far;
        const bool bad = block < 0 || block >= a.cache.num_blocks;  // reported, and read as zeros
        if (j < n && bad) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        if (!ready && at + n >= row_end) {  // the row's last block
            pkv::pdl_wait();
            ready = true;
        }
        const int stage = issued % kStages;
        if (issued >= kStages) {
            ok = wait_bounded(pkv::smem_addr(&empty[stage]), (issued / kStages - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;  // a consumer gave up
        }
        const uint32_t dst = ring + stage * kStageBytes, bar = pkv::smem_addr(&full[stage]);
        if (lane == 0) pkv::mbar_arrive_expect_tx(bar, n * kBlockTraffic);
        __syncwarp();
        if (j < n && lane < 16) {
            const int64_t tile = layer_tile + static_cast<int64_t>(block) * kHeads;
            if (lane < 8) {
                const uint8_t *codes = lane < 4 ? a.cache.key_codes : a.cache.value_codes;
                bulk_load(dst + (lane < 4 ? j * kBlockBytes : kValueAt + j * kValuePitch),
                          bad ? kZeroTiles : codes + tile * kTile, kBlockBytes, bar, policy);
            } else {
                const float *scales = lane < 12 ? a.cache.key_scales : a.cache.value_scales;
                bulk_load(dst + kScaleAt + (lane < 12 ? j : kChunk + j) * 16, bad ? kLeastScales : scales + tile, 16, bar,
                          policy);
            }
        }
        at += n;
        ++issued;
    }
    if (!ok && lane == 0) atomicOr(a.error_flag, PKV_DEVICE_WAIT_TIMEOUT);
    // No copy may land after the CTA has left.
    for (int c = max(0, issued - kStages); c < issued; ++c) {
        wait_bounded(pkv::smem_addr(&full[c % kStages]), (c / kStages) & 1);
    }
    if (!ready) pkv::pdl_wait();
}

template <bool SPLIT_Q>
__global__ void __launch_bounds__(kThreads, 3) fp8_decode_kernel(const __grid_constant__ Args a) {
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
    // Launched as a programmatic dependent: behind the append of the same layer
    // (early) the tables and every block but the rows' last ones are ready, and only
    // what the append writes is waited for.
    bool ready = !a.early;
    if (ready) pkv::pdl_wait();

    // The piece, and a first cut of the rows: 32 samples of prefix, `step` rows apart.
    int step = (a.batch + 31) / 32;
    int sample = lane * step < a.batch ? a.prefix[min((lane + 1) * step, a.batch)] : INT32_MAX;
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
    if (total == 0 || static_cast<int>(blockIdx.x) >= pieces) {
        if (!ready) pkv::pdl_wait();
        return;
    }
    const int begin = piece_begin(blockIdx.x, total, pieces);
    const int end = piece_begin(blockIdx.x + 1, total, pieces);
    // The first row with blocks past `begin`: the first sample past it, cut finer until
    // the samples are rows.
    int lo = 0;
    while (true) {
        const unsigned past = __ballot_sync(0xffffffffu, sample > begin);
        lo += (past != 0 ? __ffs(past) - 1 : 31) * step;
        if (step <= 32) break;
        step = (step + 31) / 32;
        sample = lo + lane * step < a.batch ? a.prefix[min(lo + (lane + 1) * step, a.batch)] : INT32_MAX;
    }
    if (warp == kProducer) {
        fill_ring(a, begin, end, lo, ready, lane, smem, full, empty);
        return;
    }
    Rows rows = load_rows(a, lo, lane);
    int row = advance_row(a, rows, lo, begin, lane);
    if (!ready) pkv::pdl_wait();
    pkv::pdl_launch_dependents();

    bool beyond = row >= a.batch;  // prefix does not grow from row to row
    int row_first = __shfl_sync(0xffffffffu, rows.first, row - rows.base);
    uint32_t q[8];
    const uint32_t low = pkv::smem_addr(smem) + kLowAt + threadIdx.x * 32;
    if (!beyond) load_query<SPLIT_Q>(a, row, warp * kGroup + g, t, q, low);

    int consumed = 0;
    bool failed = false;
    int i = begin;
    while (i < end && !beyond) {
        const int row_last = __shfl_sync(0xffffffffu, rows.last, row - rows.base);
        const int length = __shfl_sync(0xffffffffu, rows.length, row - rows.base);
        const int seg_end = min(end, row_last);
        // The next row's query is brought near while this row streams.
        int row_next = row;
        Rows rows_next = rows;
        if (row_last < end) {
            row_next = advance_row(a, rows_next, row + 1, row_last, lane);
            beyond = row_next >= a.batch;
            if (!beyond) prefetch_query<SPLIT_Q>(a, row_next, warp * kGroup + g, t);
        }

        float m0 = kLowest, m1 = kLowest, l0 = 0.f, l1 = 0.f;
        float o[4][4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;

        while (i < seg_end) {
            const int n = min(kChunk, seg_end - i);
            const int stage = consumed % kStages;
            const uint8_t *src = smem + stage * kStageBytes;
            failed = !wait_bounded(pkv::smem_addr(&full[stage]), (consumed / kStages) & 1);
            failed = __any_sync(0xffffffffu, failed);
            if (failed) break;
            const int tokens = min(max(length - (i - row_first) * kSlots, 0), n * kSlots);  // valid ones of the chunk

            // Scores: lane's rows are tokens 4 j + (g & 1) and 4 j + 2 + (g & 1) of block g / 2.
            float s[4][4];
            const uint8_t *k_at = src + (g >> 1) * kBlockBytes + warp * kTile + (g & 1) * kDim + 16 * t;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 a0 = *reinterpret_cast<const uint4 *>(k_at + 4 * j * kDim);
                const uint4 a1 = *reinterpret_cast<const uint4 *>(k_at + (4 * j + 2) * kDim);
                s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const uint32_t x = word(a0, ks), y = word(a1, ks);
                    uint32_t k0, k1, k2, k3;
                    pkv::fp8::decode4(x, k0, k2);
                    pkv::fp8::decode4(y, k1, k3);
                    mma(s[j], k0, k1, k2, k3, q[2 * ks], q[2 * ks + 1]);
                    if (SPLIT_Q) {
                        const uint2 half = lds64(low + 8 * ks);
                        mma(s[j], k0, k1, k2, k3, half.x, half.y);
                    }
                }
            }
            const float key_scale =
                *reinterpret_cast<const float *>(src + kScaleAt + (g >> 1) * 16 + warp * 4) * (SPLIT_Q ? 2.f : 1.f) * kScaleLog2;
            const float value_scale =
                *reinterpret_cast<const float *>(src + kScaleAt + (kChunk + (g >> 1)) * 16 + warp * 4);
            uint4 v[4][2];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const uint8_t *v_at = src + kValueAt + t * kValuePitch + warp * kTile + (16 * mt + g) * 16;
                v[mt][0] = *reinterpret_cast<const uint4 *>(v_at);
                v[mt][1] = *reinterpret_cast<const uint4 *>(v_at + 8 * 16);
            }
            // Every lane has read the stage (the fence orders the reads before the
            // copies, the warp barrier the lanes): it may be filled again while this
            // chunk is worked on.
            pkv::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) pkv::mbar_arrive(pkv::smem_addr(&empty[stage]));
            i += n;
            ++consumed;

            const int ve = ((__float_as_int(value_scale) >> 23) & 0xff) - 127;
            const float shift = static_cast<float>(ve);
            const float unscale = pkv::fp8::exp2_int(-ve);
            // Blocks past n hold an earlier chunk's bytes: their tokens are masked below.
            const bool whole = tokens == kChunk * kSlots;
            float top0 = kLowest, top1 = kLowest;
            const int held = tokens - (g >> 1) * kSlots;  // valid tokens from block g / 2 on
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j][0] = fmaf(s[j][0], key_scale, shift);
                s[j][1] = fmaf(s[j][1], key_scale, shift);
                s[j][2] = fmaf(s[j][2], key_scale, shift);
                s[j][3] = fmaf(s[j][3], key_scale, shift);
                if (!whole) {
                    const int token = 4 * j + (g & 1);
                    if (token >= held) s[j][0] = s[j][1] = -INFINITY;
                    if (token + 2 >= held) s[j][2] = s[j][3] = -INFINITY;
                }
                top0 = fmaxf(top0, fmaxf(s[j][0], s[j][2]));
                top1 = fmaxf(top1, fmaxf(s[j][1], s[j][3]));
            }
            top0 = max8(top0);
            top1 = max8(top1);
            top0 = fmaxf(m0, fabsf(top0) > kFarScore ? top0 : top0 - kWeightShift);
            top1 = fmaxf(m1, fabsf(top1) > kFarScore ? top1 : top1 - kWeightShift);
            const float alpha0 = pkv::exp2_approx(m0 - top0);
            const float alpha1 = pkv::exp2_approx(m1 - top1);
            m0 = top0;
            m1 = top1;
            float add0 = 0.f, add1 = 0.f;
            uint32_t p[4][2], pl[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w0 = pkv::exp2_approx(s[j][0] - m0);
                const float w1 = pkv::exp2_approx(s[j][1] - m1);
                const float w2 = pkv::exp2_approx(s[j][2] - m0);
                const float w3 = pkv::exp2_approx(s[j][3] - m1);
                add0 += w0 + w2;
                add1 += w1 + w3;
                const __half2 h01 = __floats2half2_rn(w0, w1), h23 = __floats2half2_rn(w2, w3);
                const float2 f01 = __half22float2(h01), f23 = __half22float2(h23);
                p[j][0] = pkv::movmatrix_trans(pkv::pack_half2(h01));
                p[j][1] = pkv::movmatrix_trans(pkv::pack_half2(h23));
                pl[j][0] = pkv::movmatrix_trans(pkv::pack_half2(__floats2half2_rn(w0 - f01.x, w1 - f01.y)));
                pl[j][1] = pkv::movmatrix_trans(pkv::pack_half2(__floats2half2_rn(w2 - f23.x, w3 - f23.y)));
            }
            // A block whose tokens are all masked adds nothing, whatever its scale row holds.
            if (!whole && held <= 0) add0 = add1 = 0.f;
            else {
                add0 *= unscale;
                add1 *= unscale;
            }
            l0 = fmaf(l0, alpha0, add0);
            l1 = fmaf(l1, alpha1, add1);
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                o[mt][0] *= alpha0;
                o[mt][1] *= alpha1;
                o[mt][2] *= alpha0;
                o[mt][3] *= alpha1;
                if (!whole) {  // weight 0 times NaN is NaN
                    const int keep = tokens - t * kSlots;
                    v[mt][0] = keep_bytes(v[mt][0], keep);
                    v[mt][1] = keep_bytes(v[mt][1], keep);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = word(v[mt][0], j), y = word(v[mt][1], j);
                    uint32_t v0, v1, v2, v3;
                    pkv::fp8::decode4(x, v0, v2);
                    pkv::fp8::decode4(y, v1, v3);
                    mma(o[mt], v0, v1, v2, v3, p[j][0], p[j][1]);
                    mma(o[mt], v0, v1, v2, v3, pl[j][0], pl[j][1]);
                }
            }
        }
        if (failed) break;

        l0 = sum8(l0);
        l1 = sum8(l1);
        const int head0 = warp * kGroup + 2 * t;
        if (row_first >= begin && row_last <= end) {
            // Normalise and round; a row whose every token is masked is zeros.
            __half *dst = a.out + row * a.out_stride;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const int d = 16 * mt + g;
                dst[head0 * kDim + d] = __float2half_rn(l0 == 0.f ? 0.f : __fdiv_rn(o[mt][0], l0));
                dst[(head0 + 1) * kDim + d] = __float2half_rn(l1 == 0.f ? 0.f : __fdiv_rn(o[mt][1], l1));
                dst[head0 * kDim + d + 8] = __float2half_rn(l0 == 0.f ? 0.f : __fdiv_rn(o[mt][2], l0));
                dst[(head0 + 1) * kDim + d + 8] = __float2half_rn(l1 == 0.f ? 0.f : __fdiv_rn(o[mt][3], l1));
            }
        } else if (pieces == 1) {  // begins before the list or ends behind it
            if (lane == 0) atomicOr(a.error_flag, PKV_DEVICE_BAD_BLOCK);
        } else {
            const int64_t index = static_cast<int64_t>(row) + blockIdx.x;
            float *po = a.part_o + index * kQueryHeads * kDim;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const int d = 16 * mt + g;
                po[head0 * kDim + d] = o[mt][0];
                po[(head0 + 1) * kDim + d] = o[mt][1];
                po[head0 * kDim + d + 8] = o[mt][2];
                po[(head0 + 1) * kDim + d + 8] = o[mt][3];
            }
            if (g == 0) {
                *reinterpret_cast<float4 *>(a.part_ml + index * kQueryHeads * 2 + head0 * 2) = make_float4(m0, l0, m1, l1);
            }
        }
        if (row_last < end) {
            row = row_next;
            rows = rows_next;
            row_first = row_last;
            if (!beyond) load_query<SPLIT_Q>(a, row, warp * kGroup + g, t, q, low);
        }
    }
    if ((failed || beyond) && lane == 0) {
        atomicOr(a.error_flag, failed ? PKV_DEVICE_WAIT_TIMEOUT : PKV_DEVICE_BAD_BLOCK);
    }
}

// Merge of the rows that several pieces hold, sixteen lanes a head and four dims
// a lane.  With few rows a CTA's eight warps deal out the pieces of one (row, two
// heads) and the first warp merges the warps' results in order, so a row of 32
// pieces is four dependent loads deep; with many rows a warp merges a row's few
// pieces.
constexpr int kMergeWarps = 8;
constexpr int kMergeThreads = kMergeWarps * 32;

template <bool SPREAD>
__global__ void __launch_bounds__(kMergeThreads) fp8_merge_kernel(const __grid_constant__ Args a) {
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

// The rotated queries of pkv_fp8_decode_layer (all high halves, then all low ones), then the partials.
constexpr int64_t kQueryRowBytes = 2 * kQueryHeads * kDim * 2;

int64_t workspace_of(int64_t batch, int64_t grid) {
    return batch * kQueryRowBytes + (grid > 1 ? (batch + grid) * kPartial * 4 : 0);
}

struct DeviceInfo {
    int sms = 0;
    int ctas_per_sm = 0;
};

cudaError_t prepare_kernel(void (*kernel)(Args), int *ctas_per_sm) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas_per_sm, kernel, kThreads, kSmem);
    return e;
}

constexpr int kMaxDevices = 64;

// SMs and resident CTAs of `device`, found out (and the kernels' attributes set) at its first use.
int device_info(int device, DeviceInfo *info) {
    static std::atomic<int> sms[kMaxDevices] = {}, ctas[kMaxDevices] = {};
    const bool known = device >= 0 && device < kMaxDevices;
    if (known && ctas[device].load(std::memory_order_acquire) > 0) {
        info->sms = sms[device].load(std::memory_order_relaxed);
        info->ctas_per_sm = ctas[device].load(std::memory_order_relaxed);
        return PKV_OK;
    }
    int previous = 0, plain = 0, split = 0;
    cudaError_t e = cudaGetDevice(&previous);
    if (e == cudaSuccess) e = cudaSetDevice(device);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 decode: ") + cudaGetErrorString(e));
    e = cudaDeviceGetAttribute(&info->sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = prepare_kernel(fp8_decode_kernel<false>, &plain);
    if (e == cudaSuccess) e = prepare_kernel(fp8_decode_kernel<true>, &split);
    // The merge keeps the split kernel's partition of L1 and shared memory.
    for (const auto merge : {fp8_merge_kernel<false>, fp8_merge_kernel<true>}) {
        if (e == cudaSuccess) {
            e = cudaFuncSetAttribute(merge, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        }
    }
    cudaSetDevice(previous);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 decode: ") + cudaGetErrorString(e));
    const int least = plain < split ? plain : split;
    info->ctas_per_sm = least < 1 ? 1 : least;
    if (known) {
        sms[device].store(info->sms, std::memory_order_relaxed);
        ctas[device].store(info->ctas_per_sm, std::memory_order_release);
    }
    return PKV_OK;
}

}  // namespace

extern "C" int pkv_fp8_decode_plan(int32_t device, int32_t batch, int32_t total_blocks, int32_t *out_grid,
                                   int64_t *out_workspace_bytes) {
    pkv::clear_error();
    if (out_grid == nullptr || out_workspace_bytes == nullptr || batch < 1 || total_blocks < 0) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 decode plan: needs a nonempty batch");
    }
    DeviceInfo info;
    const int rc = device_info(device, &info);
    if (rc) return rc;
    const int grid = pieces_of(total_blocks, info.sms * info.ctas_per_sm);  // at most one CTA per resident slot
    *out_grid = grid;
    *out_workspace_bytes = workspace_of(batch, grid);
    return PKV_OK;
}

namespace {

// The attention of pkv_fp8_decode_attention, with the append of pkv_fp8_decode_layer before it when `key` is given.
int decode(const pkv::fp8::Cache &cache, int32_t layer, const void *query, int64_t query_stride, const void *key,
           const void *value, int64_t kv_stride, const void *rope_table, bool clear, const int32_t *lengths,
           const int32_t *prefix, const int32_t *flat, int32_t batch, int32_t total_blocks, int32_t grid, void *out,
           int64_t out_stride, void *workspace, int64_t workspace_bytes, int32_t *error_flag, cudaStream_t stream) {
    int rc = pkv::fp8::check_cache(cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales,
                                   cache.layers, cache.num_blocks, layer, 1);
    if (rc) return rc;
    if (query == nullptr || lengths == nullptr || prefix == nullptr || (flat == nullptr && total_blocks > 0) ||
        out == nullptr || error_flag == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 decode: null pointer argument");
    }
    if (batch < 1 || total_blocks < 0 || grid < 1) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 decode: batch, block count or grid out of range");
    }
    if ((reinterpret_cast<uintptr_t>(query) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) || query_stride % 8 ||
        out_stride % 8 || query_stride < kQueryHeads * kDim || out_stride < kQueryHeads * kDim) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 decode: rows must be 16-byte aligned, 2048 or more values apart in multiples of 8");
    }
    const int64_t slots = static_cast<int64_t>(batch) + grid;
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < workspace_of(batch, grid)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 decode: the workspace is too small (see pkv_fp8_decode_plan)");
    }
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
    DeviceInfo info;
    if ((rc = device_info(device, &info))) return rc;
    const __half *query_low = nullptr;
    if (key != nullptr) {
        __half *const low = static_cast<__half *>(workspace) + static_cast<int64_t>(batch) * kQueryHeads * kDim;
        query_low = low;
        rc = pkv::fp8::launch_decode_append(cache, layer, key, value, kv_stride, rope_table, query, query_stride, workspace, low,
                                            lengths, prefix, flat, batch, total_blocks, error_flag, stream);
        if (rc) return rc;
        query = workspace;
        query_stride = kQueryHeads * kDim;
    }
    float *const partials = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + batch * kQueryRowBytes);
    Args a;
    a.cache = cache;
    a.layer = layer;
    a.query = static_cast<const __half *>(query);
    a.query_low = query_low;
    a.query_stride = query_stride;
    a.lengths = lengths;
    a.prefix = prefix;
    a.flat = flat;
    a.batch = batch;
    a.capacity = total_blocks;
    a.grid = grid;
    a.clear = clear;
    a.early = key != nullptr;
    a.out = static_cast<__half *>(out);
    a.out_stride = out_stride;
    a.part_o = partials;
    a.part_ml = partials + slots * kQueryHeads * kDim;
    a.error_flag = error_flag;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    e = cudaLaunchKernelEx(&config, key != nullptr ? fp8_decode_kernel<true> : fp8_decode_kernel<false>, a);
    if (e == cudaSuccess && grid > 1) {
        // A CTA per (row, two heads) while that is at most two waves of CTAs: beyond it rows
        // have few pieces each and a warp merges them as fast.
        const int64_t pairs = static_cast<int64_t>(batch) * (kQueryHeads / 2);
        const bool spread = pairs <= 16 * info.sms;
        const auto blocks = static_cast<unsigned>(spread ? pairs : (pairs + kMergeWarps - 1) / kMergeWarps);
        e = pkv::launch_pdl(spread ? fp8_merge_kernel<true> : fp8_merge_kernel<false>, dim3(blocks), dim3(kMergeThreads),
                            config.stream, a);
    }
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 decode launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

// The same with the append before it; clear: rows without blocks give zeros.
int decode_layer(const pkv::fp8::Cache &cache, int32_t layer, const void *query, int64_t query_stride, const void *key,
                 const void *value, int64_t kv_stride, const void *rope_table, bool clear, const int32_t *lengths,
                 const int32_t *prefix, const int32_t *flat, int32_t batch, int32_t total_blocks, int32_t grid, void *out,
                 int64_t out_stride, void *workspace, int64_t workspace_bytes, int32_t *error_flag, cudaStream_t stream) {
    pkv::clear_error();
    if (key == nullptr || value == nullptr || rope_table == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 decode layer: key, value and rope_table are required");
    }
    return decode(cache, layer, query, query_stride, key, value, kv_stride, rope_table, clear, lengths, prefix, flat,
                  batch, total_blocks, grid, out, out_stride, workspace, workspace_bytes, error_flag, stream);
}

}  // namespace

extern "C" int pkv_fp8_decode_attention(const void *key_codes, const void *value_codes, const void *key_scales,
                                        const void *value_scales, int32_t layers, int32_t num_blocks, int32_t layer,
                                        const void *query, int64_t query_stride, const int32_t *lengths,
                                        const int32_t *prefix, const int32_t *flat, int32_t batch, int32_t total_blocks,
                                        int32_t grid, void *out, int64_t out_stride, void *workspace,
                                        int64_t workspace_bytes, int32_t *error_flag, void *stream) {
    pkv::clear_error();
    return decode(pkv::fp8::cache_of(key_codes, value_codes, key_scales, value_scales, layers, num_blocks), layer, query,
                  query_stride, nullptr, nullptr, 0, nullptr, true, lengths, prefix, flat, batch, total_blocks, grid,
                  out, out_stride, workspace, workspace_bytes, error_flag, static_cast<cudaStream_t>(stream));
}

extern "C" int pkv_fp8_decode_layer(void *key_codes, void *value_codes, void *key_scales, void *value_scales,
                                    int32_t layers, int32_t num_blocks, int32_t layer, const void *query,
                                    int64_t query_stride, const void *key, const void *value, int64_t kv_stride,
                                    const void *rope_table, const int32_t *lengths, const int32_t *prefix,
                                    const int32_t *flat, int32_t batch, int32_t total_blocks, int32_t grid, void *out,
                                    int64_t out_stride, void *workspace, int64_t workspace_bytes, int32_t *error_flag,
                                    void *stream) {
    return decode_layer(pkv::fp8::cache_of(key_codes, value_codes, key_scales, value_scales, layers, num_blocks), layer, query,
                        query_stride, key, value, kv_stride, rope_table, false, lengths, prefix, flat, batch, total_blocks,
                        grid, out, out_stride, workspace, workspace_bytes, error_flag, static_cast<cudaStream_t>(stream));
}

extern "C" int pkv_fp8_decode_layer_zero(void *key_codes, void *value_codes, void *key_scales, void *value_scales,
                                         int32_t layers, int32_t num_blocks, int32_t layer, const void *query,
                                         int64_t query_stride, const void *key, const void *value, int64_t kv_stride,
                                         const void *rope_table, const int32_t *lengths, const int32_t *prefix,
                                         const int32_t *flat, int32_t batch, int32_t total_blocks, int32_t grid, void *out,
                                         int64_t out_stride, void *workspace, int64_t workspace_bytes, int32_t *error_flag,
                                         void *stream) {
    return decode_layer(pkv::fp8::cache_of(key_codes, value_codes, key_scales, value_scales, layers, num_blocks), layer, query,
                        query_stride, key, value, kv_stride, rope_table, true, lengths, prefix, flat, batch, total_blocks,
                        grid, out, out_stride, workspace, workspace_bytes, error_flag, static_cast<cudaStream_t>(stream));
}
