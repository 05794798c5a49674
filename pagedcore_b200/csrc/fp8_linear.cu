// 8-bit linear layer on the sm_100a tensor cores:
//   y[m][n] = fp16( sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] * w[n][k] )
// with E4M3 codes x [rows][k] and w [n][k] and FP32 scales per row of x and
// 128 values, and per 128 x 128 block of w.
//
// To 64 rows the weight is the MMA's M side (128 weight rows a tile) and the rows
// of x its N side (all of them one tile of NT = 16, 32 or 64): at decode the weight
// is the large operand and is read once.  (More rows: the two kernels below.)  One K block of 128 is four tcgen05.mma (kind::f8f6f4, K = 32)
// into a TMEM buffer of its own; the scales differ from block to block, so a
// block's sums are read back and added into FP32 registers times sx * sw (sw is
// one number for the tile and block, sx one per column).  Two TMEM buffers let
// the tensor cores work on the next block meanwhile.
//
// Work split: one CTA per 128 weight rows; where that leaves
// SMs idle the K blocks of a tile are dealt to the 2, 4 or 8 CTAs of a cluster,
// which add their FP32 sums through distributed shared memory in rank order and
// write FP16: one launch, and results that do not depend on timing.
//
// Roles: warps 0 to 3 read TMEM, scale and add (warp w lanes 32 w ..); warp 4
// loads by TMA (one 128-byte swizzled box of each operand a stage, no multicast);
// warp 5 owns the TMEM allocation and issues the MMAs.  Every wait is bounded; one that
// runs out sets PKV_DEVICE_WAIT_TIMEOUT, and the CTA goes on without waiting so
// that no barrier is left short.

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "pagedkv.h"
#include "ptx.cuh"
#include "status.h"
#include "tcgen05.cuh"
#include "tensor_maps.h"

namespace {

constexpr int kTileRows = 128;  // weight rows a tile: MMA M, and the height of a weight scale's block
constexpr int kKBlock = 128;    // values a scale covers: one 128-byte swizzle row
constexpr int kWBytes = kTileRows * kKBlock;
constexpr uint32_t kWaitPolls = 1u << 24;
constexpr int kMaxCluster = 8;

// The kernel for few rows: NT rows of x, at most 64.
template <int NT>
struct Shape {
    static constexpr int kEpilogueWarps = 4;
    static constexpr int kThreads = (kEpilogueWarps + 2) * 32;
    static constexpr int kColumns = NT;  // of one epilogue warp
    static constexpr int kStageBytes = kWBytes + NT * kKBlock;
    static constexpr int kStages = 4;
    static constexpr int kTmemColumns = 2 * NT < 32 ? 32 : 2 * NT;
    // The ring, reused at the end for [NT][128] FP32 sums.
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kSums = NT * kTileRows * 4;
    static constexpr int kSmem = (kRing > kSums ? kRing : kSums) + 1024;
};

struct LinearArgs {
    const float *x_scales;  // [rows][k_blocks]
    const float *w_scales;  // [ceil(n / 128)][k_blocks]
    __half *out;
    int64_t out_stride;
    int32_t rows;
    int32_t n;
    int32_t k_blocks;
    int32_t splits;   // CTAs of a cluster
    int32_t n_tiles;
    int32_t m_tiles;     // many rows: tiles of 128 rows of x
    int32_t tiles;       // many rows: all
    int32_t w_blocks;    // ceil(n / 128)
    int32_t vector_out;  // rows of out take 16-byte stores
    int32_t *error_flag;
};

__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, int32_t *error_flag) {
    if (pkv::mbar_test_wait(bar, parity) || pkv::mbar_wait_bounded(bar, parity, kWaitPolls)) return true;
    atomicOr(error_flag, PKV_DEVICE_WAIT_TIMEOUT);
    return false;
}

// D[tmem] (+)= A[smem] . B[smem]^T, E4M3 operands, FP32 D (one thread).
__device__ __forceinline__ void mma_f8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          bool accumulate) {
    const uint32_t acc = accumulate ? 1u : 0u;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}

// Instruction descriptor of kind::f8f6f4: FP32 D, E4M3 A and B (format 0), both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) {
    return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// This CTA's shared-memory address as seen in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr));
    return v;
}

// The sum over the cluster's CTAs of the four FP32 values at `addr`, in rank
// order; every rank's load is under way before the first is used.
__device__ __forceinline__ float4 cluster_sum(uint32_t addr, int splits) {
    float4 part[kMaxCluster];
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
        if (s < splits) part[s] = ld_cluster_f4(map_to_rank(addr, s));
    }
    float4 v = part[0];
#pragma unroll
    for (int s = 1; s < kMaxCluster; ++s) {
        if (s < splits) v.x += part[s].x, v.y += part[s].y, v.z += part[s].z, v.w += part[s].w;
    }
    return v;
}

// Bring a box into L2 (a hint: no data is used, so nothing has to be waited for first).
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap *map, int32_t c0, int32_t c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1)
                 : "memory");
}

// Four outputs of row m at column n (a multiple of 4), rounded to FP16.
__device__ __forceinline__ void store4(const LinearArgs &a, int m, int n, const float4 &v) {
    __half *dst = a.out + static_cast<int64_t>(m) * a.out_stride + n;
    if (a.vector_out && n + 4 <= a.n) {
        uint2 h;
        h.x = pkv::pack_half2(__floats2half2_rn(v.x, v.y));
        h.y = pkv::pack_half2(__floats2half2_rn(v.z, v.w));
        *reinterpret_cast<uint2 *>(dst) = h;
    } else {
        if (n < a.n) dst[0] = __float2half_rn(v.x);
        if (n + 1 < a.n) dst[1] = __float2half_rn(v.y);
        if (n + 2 < a.n) dst[2] = __float2half_rn(v.z);
        if (n + 3 < a.n) dst[3] = __float2half_rn(v.w);
    }
}

template <int NT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 2)
    fp8_linear_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                      const LinearArgs a) {
    using S = Shape<NT>;
    extern __shared__ uint8_t dyn_smem[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], tmem_full[2], tmem_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float factors[2][NT];  // sx * sw of the current K block's columns

    const uint32_t raw = pkv::smem_addr(dyn_smem);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const int split = static_cast<int>(blockIdx.x) % a.splits;  // rank in the cluster
    const int n_tile = static_cast<int>(blockIdx.x) / a.splits;
    const int n0 = n_tile * kTileRows;
    constexpr int m0 = 0;  // all rows are one tile
    const int kb_begin = static_cast<int>(static_cast<int64_t>(split) * a.k_blocks / a.splits);
    const int kb_end = static_cast<int>(static_cast<int64_t>(split + 1) * a.k_blocks / a.splits);
    const int count = kb_end - kb_begin;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    constexpr int kProducer = S::kEpilogueWarps;
    constexpr int kMma = S::kEpilogueWarps + 1;

    if (warp == kMma) {
        pkv::tc::tmem_alloc(pkv::smem_addr(&tmem_slot), S::kTmemColumns);
        pkv::tc::tmem_relinquish();
    }
    if (threadIdx.x == kProducer * 32) {
        for (int s = 0; s < S::kStages; ++s) {
            pkv::mbar_init(pkv::smem_addr(&full[s]), 1);
            pkv::mbar_init(pkv::smem_addr(&empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            pkv::mbar_init(pkv::smem_addr(&tmem_full[b]), 1);
            pkv::mbar_init(pkv::smem_addr(&tmem_empty[b]), S::kEpilogueWarps);
        }
        pkv::fence_barrier_init();
    }
    pkv::tc::fence_before_sync();
    __syncthreads();
    pkv::tc::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pkv::pdl_launch_dependents();

    float acc[S::kColumns];
#pragma unroll
    for (int c = 0; c < S::kColumns; ++c) acc[c] = 0.f;

    if (warp == kProducer) {
        int issued = 0;
        if (lane == 0) {
            const uint64_t reused = pkv::l2_policy_evict_last();
            // The weight's first boxes start towards L2 while the kernel before this one ends.
            for (int i = 0; i < min(count, S::kStages); ++i) tma_prefetch_2d(&w_map, (kb_begin + i) * kKBlock, n0);
            pkv::pdl_wait();
            for (int i = 0; i < count; ++i) {
                const int st = i % S::kStages;
                if (i >= S::kStages &&
                    !wait_bounded(pkv::smem_addr(&empty[st]), ((i / S::kStages) - 1) & 1, a.error_flag)) {
                    break;
                }
                issued = i + 1;
                const uint32_t bar = pkv::smem_addr(&full[st]);
                pkv::mbar_arrive_expect_tx(bar, S::kStageBytes);
                pkv::tma_load_2d(base + st * S::kStageBytes, &w_map, (kb_begin + i) * kKBlock, n0, bar);
                pkv::tma_load_2d_hint(base + st * S::kStageBytes + kWBytes, &x_map, (kb_begin + i) * kKBlock, m0, bar,
                                      reused);
            }
            // No copy may land once the ring is reused or the CTA has left.
            for (int i = max(0, issued - S::kStages); i < issued; ++i) {
                pkv::mbar_wait_bounded(pkv::smem_addr(&full[i % S::kStages]), (i / S::kStages) & 1, kWaitPolls);
            }
        } else {
            pkv::pdl_wait();
        }
    } else if (warp == kMma) {
        pkv::pdl_wait();
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_e4m3_f32(kTileRows, NT);
            for (int i = 0; i < count; ++i) {
                const int st = i % S::kStages;
                const int buf = i & 1;
                if (!wait_bounded(pkv::smem_addr(&full[st]), (i / S::kStages) & 1, a.error_flag)) break;
                if (i >= 2 && !wait_bounded(pkv::smem_addr(&tmem_empty[buf]), ((i >> 1) - 1) & 1, a.error_flag)) break;
                pkv::tc::fence_after_sync();
                const uint32_t w_src = base + st * S::kStageBytes;
#pragma unroll
                for (int k = 0; k < kKBlock / 32; ++k) {
                    mma_f8_ss(tmem + buf * NT, pkv::tc::desc_k_major_sw128(w_src + 32 * k),
                              pkv::tc::desc_k_major_sw128(w_src + kWBytes + 32 * k), idesc, k > 0);
                }
                pkv::tc::commit(pkv::smem_addr(&empty[st]));
                pkv::tc::commit(pkv::smem_addr(&tmem_full[buf]));
            }
        }
        __syncwarp();
    } else {
        pkv::pdl_wait();
        constexpr int kEpilogueThreads = S::kEpilogueWarps * 32;
        // Thread c < NT loads column c's scale two K blocks ahead; the two factors
        // stay apart until they are used, so that nothing waits for a load.
        const int column = m0 + static_cast<int>(threadIdx.x);
        const bool loads = threadIdx.x < NT;
        const bool inside = loads && column < a.rows;
        const float *sx = a.x_scales + static_cast<int64_t>(inside ? column : 0) * a.k_blocks + kb_begin;
        const float *sw = a.w_scales + static_cast<int64_t>(n_tile) * a.k_blocks + kb_begin;
        float x0 = inside ? sx[0] : 0.f, w0 = sw[0];
        float x1 = inside && count > 1 ? sx[1] : 0.f, w1 = count > 1 ? sw[1] : 0.f;
        const int first = (warp >> 2) * S::kColumns;  // of this warp's columns
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        bool ok = true;
        for (int i = 0; i < count; ++i) {
            const int buf = i & 1;
            if (loads) factors[buf][threadIdx.x] = x0 * w0;
            x0 = x1;
            w0 = w1;
            if (i + 2 < count) {
                if (inside) x1 = sx[i + 2];
                w1 = sw[i + 2];
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory");
            if (ok) ok = wait_bounded(pkv::smem_addr(&tmem_full[buf]), (i >> 1) & 1, a.error_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                pkv::tc::fence_after_sync();
                constexpr int kStep = S::kColumns < 32 ? S::kColumns : 32;
#pragma unroll
                for (int c = 0; c < S::kColumns; c += kStep) {
                    uint32_t d[kStep];
                    if constexpr (kStep == 32) {
                        pkv::tc::tmem_ld32(tmem + lanes + buf * NT + first + c, d);
                    } else {
                        pkv::tc::tmem_ld16(tmem + lanes + buf * NT + first + c, d);
                    }
                    pkv::tc::tmem_wait_ld();
                    const float4 *f = reinterpret_cast<const float4 *>(&factors[buf][first + c]);
#pragma unroll
                    for (int j = 0; j < kStep / 4; ++j) {
                        const float4 s = f[j];
                        acc[c + 4 * j] = fmaf(__uint_as_float(d[4 * j]), s.x, acc[c + 4 * j]);
                        acc[c + 4 * j + 1] = fmaf(__uint_as_float(d[4 * j + 1]), s.y, acc[c + 4 * j + 1]);
                        acc[c + 4 * j + 2] = fmaf(__uint_as_float(d[4 * j + 2]), s.z, acc[c + 4 * j + 2]);
                        acc[c + 4 * j + 3] = fmaf(__uint_as_float(d[4 * j + 3]), s.w, acc[c + 4 * j + 3]);
                    }
                }
                pkv::tc::fence_before_sync();
            }
            __syncwarp();
            if (lane == 0) pkv::mbar_arrive(pkv::smem_addr(&tmem_empty[buf]));
        }
    }
    __syncthreads();  // every copy has landed and every MMA has been read (or given up on)

    // Sums as [column][128 weight rows] FP32 in the ring.
    float *sums = reinterpret_cast<float *>(dyn_smem + (base - raw));
    if (warp < S::kEpilogueWarps) {
        const int first = (warp >> 2) * S::kColumns;
        const int r = (warp & 3) * 32 + lane;
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) sums[(first + c) * kTileRows + r] = acc[c];
    }
    if (a.splits > 1) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    // Rank r adds and writes columns r, r + splits, ...: four weight rows a thread.
    const int columns = min(NT, a.rows);
    for (int item = threadIdx.x;; item += S::kThreads) {
        const int c = split + a.splits * (item / (kTileRows / 4)), r = 4 * (item % (kTileRows / 4));
        if (c >= columns) break;
        const uint32_t at = static_cast<uint32_t>((c * kTileRows + r) * 4);
        store4(a, m0 + c, n0 + r,
               a.splits == 1 ? *reinterpret_cast<const float4 *>(reinterpret_cast<const uint8_t *>(sums) + at)
                             : cluster_sum(base + at, a.splits));
    }
    if (a.splits > 1) {  // no CTA leaves while another reads its sums
        cluster_arrive();
        cluster_wait();
    }
    if (warp == kMma) {
        pkv::tc::fence_after_sync();
        pkv::tc::tmem_dealloc(tmem, S::kTmemColumns);
    }
}

// ---------------------------------------------------------------------------
// Many rows: the rows of x are the MMA's M side (128 a tile), N weight rows its N
// side.  Lane = row of x, so a thread's scale factor for a K block is one number,
// sx[row] * sw[block of its 64 columns]: no factor goes through shared memory, and
// the scaled sum is one packed FMA for two columns.  Each epilogue warp holds 64
// columns in registers (N / 16 warps, four to twelve), enough warps to cover the
// latency of the TMEM reads.  With one split the CTAs are persistent: the loads and
// MMAs of the next tile run while the last one is rounded and stored.
// ---------------------------------------------------------------------------
template <int N>
struct RowsShape {
    static constexpr int kEpilogueWarps = N / 16;
    static constexpr int kThreads = (kEpilogueWarps + 3) * 32;
    static constexpr int kXBytes = kTileRows * kKBlock;
    static constexpr int kStageBytes = kXBytes + N * kKBlock;
    static constexpr int kStages = N == 192 ? 5 : N == 128 ? 6 : 8;
    static constexpr int kBuffers = N > 128 ? 2 : 4;  // TMEM buffers
    static constexpr int kBufferColumns = N > 128 ? 256 : N;
    static constexpr int kTmemColumns = kBuffers * kBufferColumns;
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kPitch = N + 4;  // floats between the rows of a cluster's sums (in the ring)
    static_assert(kTileRows * kPitch * 4 <= kRing, "the sums fit the ring");
    static constexpr int kStoreBytes = 32 * 64;  // a warp's staging: 32 rows of 32 FP16 values
    static constexpr int kSmem = kRing + kEpilogueWarps * kStoreBytes + 1024;
};

// v[j] = p[at + j] for the indexes below `count`.  (Plain loads: the kernel before this one,
// which writes the scales of x, may still run while this one is set up.)
__device__ __forceinline__ void load_group(const float *p, int at, int count, float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = at + j < count ? p[at + j] : 0.f;
}

// acc[j] += (d[2 j], d[2 j + 1]) * f for 32 columns.
__device__ __forceinline__ void add_scaled(uint64_t *acc, const uint32_t (&d)[32], uint64_t f) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        acc[j] = pkv::fma_f32x2(pkv::f32x2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])), f, acc[j]);
    }
}

// A warp's 32 rows x 64 columns of sums (row = lane, `acc` two columns a pair)
// rounded and stored at row m, column n: 32 columns at a time through the warp's
// own 2 KiB of shared memory (16-byte chunk c of row r at chunk c ^ (r / 2 % 4): no
// bank conflicts), then 64 bytes a row.
__device__ __forceinline__ void store_rows(const LinearArgs &a, const uint64_t *acc, uint32_t staging, int m, int n,
                                           int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = pkv::unpack_f32x2(acc[16 * h + 4 * c + j]);
                w[j] = pkv::pack_half2(__floats2half2_rn(v.x, v.y));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staging + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int part = 0; part < 4; ++part) {
            const int r = part * 8 + (lane >> 2), c = lane & 3;
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(staging + r * 64 + ((c ^ ((r >> 1) & 3)) << 4))
                         : "memory");
            const int at = n + 32 * h + 8 * c;
            if (m + r < a.rows && at < a.n) {
                __half *dst = a.out + static_cast<int64_t>(m + r) * a.out_stride + at;
                if (a.vector_out && at + 8 <= a.n) {
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    const __half *v = reinterpret_cast<const __half *>(w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (at + j < a.n) dst[j] = v[j];
                    }
                }
            }
        }
        __syncwarp();
    }
}

template <int N>
__global__ void __launch_bounds__(RowsShape<N>::kThreads, 1)
    fp8_linear_rows_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                           const LinearArgs a) {
    using S = RowsShape<N>;
    extern __shared__ uint8_t dyn_smem[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], tmem_full[S::kBuffers], tmem_empty[S::kBuffers];
    __shared__ uint32_t tmem_slot;

    const uint32_t raw = pkv::smem_addr(dyn_smem);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const int split = static_cast<int>(blockIdx.x) % a.splits;
    const int first_tile = static_cast<int>(blockIdx.x) / a.splits;
    const int tile_step = static_cast<int>(gridDim.x) / a.splits;
    const int kb_begin = static_cast<int>(static_cast<int64_t>(split) * a.k_blocks / a.splits);
    const int kb_end = static_cast<int>(static_cast<int64_t>(split + 1) * a.k_blocks / a.splits);
    const int count = kb_end - kb_begin;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    constexpr int kProducer = S::kEpilogueWarps;
    constexpr int kMma = S::kEpilogueWarps + 1;

    if (warp == kMma) {
        pkv::tc::tmem_alloc(pkv::smem_addr(&tmem_slot), S::kTmemColumns);
        pkv::tc::tmem_relinquish();
    }
    if (threadIdx.x == kProducer * 32) {
        for (int s = 0; s < S::kStages; ++s) {
            pkv::mbar_init(pkv::smem_addr(&full[s]), 1);
            pkv::mbar_init(pkv::smem_addr(&empty[s]), 1);
        }
        for (int b = 0; b < S::kBuffers; ++b) {
            pkv::mbar_init(pkv::smem_addr(&tmem_full[b]), 1);
            pkv::mbar_init(pkv::smem_addr(&tmem_empty[b]), S::kEpilogueWarps);
        }
        pkv::fence_barrier_init();
    }
    pkv::tc::fence_before_sync();
    __syncthreads();
    pkv::tc::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pkv::pdl_launch_dependents();

    uint64_t acc[32];  // this warp's 64 columns, two to a register pair

    if (warp == kProducer) {
        if (lane == 0) {
            const uint64_t reused = pkv::l2_policy_evict_last();
            int issued = 0;
            bool ok = true;
            if (first_tile < a.tiles) {  // the weight's first boxes start towards L2 while the kernel before this one ends
                for (int i = 0; i < min(count, S::kStages); ++i) {
                    tma_prefetch_2d(&w_map, (kb_begin + i) * kKBlock, first_tile / a.m_tiles * N);
                }
            }
            pkv::pdl_wait();
            for (int tile = first_tile; ok && tile < a.tiles; tile += tile_step) {
                const int m0 = tile % a.m_tiles * kTileRows, n0 = tile / a.m_tiles * N;
                for (int i = 0; i < count; ++i) {
                    const int st = issued % S::kStages;
                    if (issued >= S::kStages &&
                        !wait_bounded(pkv::smem_addr(&empty[st]), ((issued / S::kStages) - 1) & 1, a.error_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = base + st * S::kStageBytes, bar = pkv::smem_addr(&full[st]);
                    pkv::mbar_arrive_expect_tx(bar, S::kStageBytes);
                    pkv::tma_load_2d(dst + S::kXBytes, &w_map, (kb_begin + i) * kKBlock, n0, bar);
                    pkv::tma_load_2d_hint(dst, &x_map, (kb_begin + i) * kKBlock, m0, bar, reused);
                    ++issued;
                }
            }
            // No copy may land once the ring is reused or the CTA has left.
            for (int i = max(0, issued - S::kStages); i < issued; ++i) {
                pkv::mbar_wait_bounded(pkv::smem_addr(&full[i % S::kStages]), (i / S::kStages) & 1, kWaitPolls);
            }
        } else {
            pkv::pdl_wait();
        }
        __syncwarp();
    } else if (warp >= kMma) {
        // Two issuing warps: each takes every other K block, so
        // one's waits and issue (about 200 and 50 clocks each) run beside the other's MMAs.
        pkv::pdl_wait();
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_e4m3_f32(kTileRows, N);
            int done = 0;
            bool ok = true;
            for (int tile = first_tile; ok && tile < a.tiles; tile += tile_step) {
                for (int i = 0; i < count; ++i, ++done) {
                    const int st = done % S::kStages;
                    const int buf = done % S::kBuffers;
                    if ((done & 1) != warp - kMma) continue;
                    ok = wait_bounded(pkv::smem_addr(&full[st]), (done / S::kStages) & 1, a.error_flag) &&
                         (done < S::kBuffers ||
                          wait_bounded(pkv::smem_addr(&tmem_empty[buf]), (done / S::kBuffers - 1) & 1, a.error_flag));
                    if (!ok) break;
                    pkv::tc::fence_after_sync();
                    const uint32_t src = base + st * S::kStageBytes;
#pragma unroll
                    for (int k = 0; k < kKBlock / 32; ++k) {
                        mma_f8_ss(tmem + buf * S::kBufferColumns, pkv::tc::desc_k_major_sw128(src + 32 * k),
                                  pkv::tc::desc_k_major_sw128(src + S::kXBytes + 32 * k), idesc, k > 0);
                    }
                    pkv::tc::commit(pkv::smem_addr(&empty[st]));
                    pkv::tc::commit(pkv::smem_addr(&tmem_full[buf]));
                }
            }
        }
        __syncwarp();
    } else {
        pkv::pdl_wait();
        const int quarter = warp & 3, first = (warp >> 2) * 64;  // TMEM lanes and columns of this warp
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t staging = base + S::kRing + warp * S::kStoreBytes;
        int done = 0;
        bool ok = true;
        for (int tile = first_tile; tile < a.tiles; tile += tile_step) {
            const int m0 = tile % a.m_tiles * kTileRows, n0 = tile / a.m_tiles * N;
            const int row = m0 + quarter * 32 + lane;
            const int block = min((n0 + first) / kTileRows, a.w_blocks - 1);  // columns past n are not stored
            // Scales four K blocks at a time, a group ahead: no register is touched
            // while its load is under way.
            const float *sx = a.x_scales + static_cast<int64_t>(min(row, a.rows - 1)) * a.k_blocks + kb_begin;
            const float *sw = a.w_scales + static_cast<int64_t>(block) * a.k_blocks + kb_begin;
            float x_next[4], w_next[4];
            load_group(sx, 0, count, x_next);
            load_group(sw, 0, count, w_next);
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[c] = 0;
            for (int group = 0; group < count; group += 4) {
                float f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = x_next[j] * w_next[j];
                load_group(sx, group + 4, count, x_next);
                load_group(sw, group + 4, count, w_next);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (group + j < count) {
                        const int buf = done % S::kBuffers;
                        if (ok) ok = wait_bounded(pkv::smem_addr(&tmem_full[buf]), (done / S::kBuffers) & 1, a.error_flag);
                        ok = __all_sync(0xffffffffu, ok);
                        ++done;
                        if (ok) {
                            pkv::tc::fence_after_sync();
                            const uint64_t f2 = pkv::f32x2(f[j], f[j]);
                            const uint32_t src = tmem + lanes + buf * S::kBufferColumns + first;
                            uint32_t d[2][32];
                            pkv::tc::tmem_ld32(src, d[0]);
                            pkv::tc::tmem_ld32(src + 32, d[1]);
                            pkv::tc::tmem_wait_ld();
                            pkv::tc::fence_before_sync();
                            __syncwarp();
                            if (lane == 0) pkv::mbar_arrive(pkv::smem_addr(&tmem_empty[buf]));
                            add_scaled(acc, d[0], f2);
                            add_scaled(acc + 16, d[1], f2);
                        }
                    }
                }
            }
            if (a.splits == 1) {
                store_rows(a, acc, staging, m0 + quarter * 32, n0 + first, lane);
            }
        }
    }

    if (a.splits > 1) {
        // One tile per cluster: each CTA leaves its sums in its ring, and rank r adds
        // and writes rows r, r + splits, ..., four columns a thread.
        __syncthreads();  // every copy has landed and every MMA has been read (or given up on)
        const int m0 = first_tile % a.m_tiles * kTileRows, n0 = first_tile / a.m_tiles * N;
        if (warp < S::kEpilogueWarps) {
            const uint32_t dst = base + (((warp & 3) * 32 + lane) * S::kPitch + (warp >> 2) * 64) * 4;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const float2 u = pkv::unpack_f32x2(acc[2 * c]), v = pkv::unpack_f32x2(acc[2 * c + 1]);
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 16 * c), "f"(u.x), "f"(u.y),
                             "f"(v.x), "f"(v.y)
                             : "memory");
            }
        }
        cluster_arrive();
        cluster_wait();
        const int rows = min(kTileRows, a.rows - m0);
        for (int item = threadIdx.x;; item += S::kThreads) {
            const int r = split + a.splits * (item / (N / 4)), c = 4 * (item % (N / 4));
            if (r >= rows) break;
            if (n0 + c < a.n) store4(a, m0 + r, n0 + c, cluster_sum(base + (r * S::kPitch + c) * 4, a.splits));
        }
        cluster_arrive();  // no CTA leaves while another reads its sums
        cluster_wait();
    } else {
        __syncthreads();
    }
    if (warp == kMma) {
        pkv::tc::fence_after_sync();
        pkv::tc::tmem_dealloc(tmem, S::kTmemColumns);
    }
}

// ---------------------------------------------------------------------------
// Many rows, large: pairs of CTAs (cta_group::2) on tiles of 256 rows of x by 256
// weight rows.  Each CTA loads its own 128 rows of x and half of the weight rows and
// holds the sums of its rows, so a K block costs an SM 32 KiB of L2 traffic for
// 128 x 256 outputs, half of what the kernel above takes; that traffic is what
// bounds the latter.  CTA 0 of a pair (the leader) issues the MMAs of both; the
// barriers that it waits on (full, tmem_empty) live in its shared memory and the other
// CTA's loads and epilogue signal them there, and its commits signal empty and
// tmem_full in both.  Sixteen epilogue warps, 64 columns each; persistent.  The epilogue
// bounds it, so its warps take registers from the others' warpgroup: 32 columns are under
// way at a time and nothing is spilled, and bulk stores take the tile out while the next
// one begins: 2047 x 11264 x 2048 in 49.3 us, 1.92 PFLOP/s, 2047 x 2048 x 5632 in 25.0.
// (The first without the bulk stores 51.3; 16 columns at a time within 96 registers 56.6;
// 60.4 with the scales two blocks ahead and spills.  With all 64 columns staged at once and
// five stages the first takes 47.8, the second 26.5.  Two halves of 128 columns with two
// TMEM buffers and an issuing warp each: 58.0.)
// ---------------------------------------------------------------------------
struct PairShape {
    static constexpr int kN = 256;
    static constexpr int kEpilogueWarps = 16;
    static constexpr int kThreads = (kEpilogueWarps + 4) * 32;  // the last warp only gives up its registers
    // Registers a thread: launched with, and how the warpgroups then share them.
    static constexpr int kRegisters = 96, kEpilogueRegisters = 112, kOtherRegisters = 32;
    static_assert(kEpilogueWarps * kEpilogueRegisters + 4 * kOtherRegisters <= (kEpilogueWarps + 4) * kRegisters,
                  "an increase would wait for registers that the block was not launched with");
    static constexpr int kXBytes = kTileRows * kKBlock;
    static constexpr int kStageBytes = kXBytes + kN / 2 * kKBlock;
    static constexpr int kStages = 6;
    static constexpr int kStoreBytes = 32 * 64;  // a warp's 32 rows of 64 FP16 values
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kSmem = kRing + kEpilogueWarps * kStoreBytes + 1024;
};

// Every lane may write the warp's staging again.
__device__ __forceinline__ void wait_staging(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

// A warp's 32 rows x 64 columns of sums (row = lane, `acc` two columns a pair) as FP16, 32
// columns at a time, in its staging (rows of 64 bytes with the 64-byte swizzle), from where
// a bulk tensor store takes them, the second while the warp goes on.  The store leaves out
// rows past the last, and columns in whole 16 bytes only.  The staging is free again after
// wait_staging.
__device__ __forceinline__ void store_rows_async(const CUtensorMap *map, const uint64_t *acc, uint32_t staging, int m,
                                                 int n, int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (h) wait_staging(lane);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = pkv::unpack_f32x2(acc[16 * h + 4 * c + j]);
                w[j] = pkv::pack_half2(__floats2half2_rn(v.x, v.y));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staging + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
        pkv::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                             reinterpret_cast<uint64_t>(map)),
                         "r"(n + 32 * h), "r"(m), "r"(staging)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}

__device__ __forceinline__ void mma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            bool accumulate) {
    const uint32_t acc = accumulate ? 1u : 0u;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}

// The barrier at this offset in both CTAs of the pair receives one arrival once
// the MMAs issued before have completed.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

// A box into this CTA's shared memory that completes on the leader's barrier (`bar`
// in the cluster's address space); no multicast.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, int32_t c0, int32_t c1,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__global__ void __launch_bounds__(PairShape::kThreads, 1)
    fp8_linear_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                           const __grid_constant__ CUtensorMap out_map, const LinearArgs a) {
    using S = PairShape;
    extern __shared__ uint8_t dyn_smem[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], tmem_full[2], tmem_empty[2];
    __shared__ uint32_t tmem_slot;

    const uint32_t raw = pkv::smem_addr(dyn_smem);
    const uint32_t base = (raw + 1023u) & ~1023u;  // the same offset in both CTAs
    const int rank = static_cast<int>(blockIdx.x) & 1;
    const int first_tile = static_cast<int>(blockIdx.x) >> 1;
    const int tile_step = static_cast<int>(gridDim.x) >> 1;
    const int count = a.k_blocks;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    constexpr int kProducer = S::kEpilogueWarps;
    constexpr int kMma = S::kEpilogueWarps + 1;

    if (warp == kMma) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pkv::smem_addr(&tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == kProducer * 32) {
        for (int s = 0; s < S::kStages; ++s) {
            pkv::mbar_init(pkv::smem_addr(&full[s]), 1);
            pkv::mbar_init(pkv::smem_addr(&empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            pkv::mbar_init(pkv::smem_addr(&tmem_full[b]), 1);
            pkv::mbar_init(pkv::smem_addr(&tmem_empty[b]), 2 * S::kEpilogueWarps);
        }
        pkv::fence_barrier_init();
    }
    pkv::tc::fence_before_sync();
    cluster_arrive();  // both CTAs' barriers and TMEM are ready
    cluster_wait();
    pkv::tc::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pkv::pdl_launch_dependents();

    if (warp >= kProducer) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegisters));
        if (warp == kProducer) {
            pkv::pdl_wait();
            if (lane == 0) {
                int issued = 0;
                bool ok = true;
                for (int tile = first_tile; ok && tile < a.tiles; tile += tile_step) {
                    const int m0 = tile % a.m_tiles * 256 + rank * 128, n0 = tile / a.m_tiles * S::kN + rank * 128;
                    for (int i = 0; i < count; ++i) {
                        const int st = issued % S::kStages;
                        if (issued >= S::kStages &&
                            !wait_bounded(pkv::smem_addr(&empty[st]), ((issued / S::kStages) - 1) & 1, a.error_flag)) {
                            ok = false;
                            break;
                        }
                        const uint32_t dst = base + st * S::kStageBytes;
                        if (rank == 0) pkv::mbar_arrive_expect_tx(pkv::smem_addr(&full[st]), 2 * S::kStageBytes);
                        const uint32_t bar = map_to_rank(pkv::smem_addr(&full[st]), 0);
                        tma_load_pair(dst, &x_map, i * kKBlock, m0, bar);
                        tma_load_pair(dst + S::kXBytes, &w_map, i * kKBlock, n0, bar);
                        ++issued;
                    }
                }
                // No copy may land after the CTA has left: every stage has been multiplied
                // (or, where a wait ran out, long since filled).
                for (int i = max(0, issued - S::kStages); i < issued; ++i) {
                    wait_bounded(pkv::smem_addr(&empty[i % S::kStages]), (i / S::kStages) & 1, a.error_flag);
                }
            }
            __syncwarp();
        } else {
            pkv::pdl_wait();
            if (rank == 0 && lane == 0 && warp < kMma + 2) {
                constexpr uint32_t idesc = idesc_e4m3_f32(256, S::kN);
                int done = 0;
                bool ok = true;
                for (int tile = first_tile; ok && tile < a.tiles; tile += tile_step) {
                    for (int i = 0; i < count; ++i, ++done) {
                        const int st = done % S::kStages;
                        const int buf = done & 1;
                        if (buf != warp - kMma) continue;  // two issuing warps, one per TMEM buffer
                        ok = wait_bounded(pkv::smem_addr(&full[st]), (done / S::kStages) & 1, a.error_flag) &&
                             (done < 2 || wait_bounded(pkv::smem_addr(&tmem_empty[buf]), ((done >> 1) - 1) & 1, a.error_flag));
                        if (!ok) break;
                        pkv::tc::fence_after_sync();
                        const uint32_t src = base + st * S::kStageBytes;
#pragma unroll
                        for (int k = 0; k < kKBlock / 32; ++k) {
                            mma_f8_pair(tmem + buf * 256, pkv::tc::desc_k_major_sw128(src + 32 * k),
                                        pkv::tc::desc_k_major_sw128(src + S::kXBytes + 32 * k), idesc, k > 0);
                        }
                        commit_pair(pkv::smem_addr(&empty[st]));
                        commit_pair(pkv::smem_addr(&tmem_full[buf]));
                    }
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kEpilogueRegisters));
        pkv::pdl_wait();
        const int quarter = warp & 3, first = (warp >> 2) * 64;
        const uint32_t src = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + first;
        const uint32_t empty0 = map_to_rank(pkv::smem_addr(&tmem_empty[0]), 0);
        uint64_t acc[32];
        int done = 0;
        bool ok = true;
        for (int tile = first_tile; tile < a.tiles; tile += tile_step) {
            const int m0 = tile % a.m_tiles * 256 + rank * 128, n0 = tile / a.m_tiles * S::kN;
            // Below 2^32: with more than one K block a row has 72 codes or more a scale.
            uint32_t sx = static_cast<uint32_t>(min(m0 + quarter * 32 + lane, a.rows - 1)) * count;
            uint32_t sw = static_cast<uint32_t>(min((n0 + first) / kTileRows, a.w_blocks - 1)) * count;
            float x = a.x_scales[sx], w = a.w_scales[sw];  // a K block ahead
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[c] = 0;
#pragma unroll 1
            for (int i = 1; i <= count; ++i) {
                const float f = x * w;
                const uint64_t f2 = pkv::f32x2(f, f);
                if (i < count) x = a.x_scales[++sx], w = a.w_scales[++sw];
                const int buf = done & 1;
                if (ok) ok = wait_bounded(pkv::smem_addr(&tmem_full[buf]), (done >> 1) & 1, a.error_flag);
                ok = __all_sync(0xffffffffu, ok);
                ++done;
                if (ok) {
                    pkv::tc::fence_after_sync();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t d[32];
                        pkv::tc::tmem_ld32(src + buf * 256 + 32 * c, d);
                        pkv::tc::tmem_wait_ld();
                        if (c == 1) {
                            pkv::tc::fence_before_sync();
                            __syncwarp();
                            if (lane == 0) arrive_cluster(empty0 + 8 * buf);
                        }
                        add_scaled(acc + 16 * c, d, f2);
                    }
                }
            }
            // From the thread's index anew: kept from before they would spill in the loop above.
            uint32_t thread;
            asm volatile("mov.u32 %0, %%tid.x;" : "=r"(thread));
            const int own = static_cast<int>(thread & 31), part = static_cast<int>(thread >> 5);
            const int m = tile % a.m_tiles * 256 + rank * 128 + (part & 3) * 32, n = tile / a.m_tiles * S::kN + (part >> 2) * 64;
            const uint32_t staging = base + S::kRing + part * S::kStoreBytes;
            if (m < a.rows && n < a.n) {
                wait_staging(own);
                if (a.vector_out && (n + 64 <= a.n || a.n % 8 == 0)) {
                    store_rows_async(&out_map, acc, staging, m, n, own);
                } else {
                    store_rows(a, acc, staging, m, n, own);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    pkv::tc::fence_before_sync();
    cluster_arrive();  // neither CTA leaves while the other's MMAs or arrivals need it
    cluster_wait();
    if (warp == kMma) {
        pkv::tc::fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
constexpr int kMaxDevices = 64;

// Map of an 8-bit matrix (rows `stride` bytes apart) in boxes of box_rows x 128 bytes with
// the 128-byte swizzle; what lies outside reads as zeros.
int byte_matrix_map(const void *base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t box_rows,
                    CUtensorMap *out) {
    const pkv::EncodeTiled encode = pkv::encode_fn();
    if (encode == nullptr) return pkv::fail(PKV_CUDA_ERROR, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {stride};
    const cuuint32_t box[2] = {kKBlock, box_rows};
    const cuuint32_t elem[2] = {1u, 1u};
    const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        return pkv::fail(PKV_CUDA_ERROR, "cuTensorMapEncodeTiled (8-bit matrix) failed with code " + std::to_string(int(r)));
    }
    return PKV_OK;
}

// Map of the output (16-byte aligned rows) in swizzled boxes, to store from.
int half_matrix_map(const LinearArgs &args, uint32_t box_columns, uint32_t box_rows, CUtensorMap *out) {
    const pkv::EncodeTiled encode = pkv::encode_fn();
    if (encode == nullptr) return pkv::fail(PKV_CUDA_ERROR, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(args.n), static_cast<cuuint64_t>(args.rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(args.out_stride) * 2};
    const cuuint32_t box[2] = {box_columns, box_rows};
    const cuuint32_t elem[2] = {1u, 1u};
    const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, args.out, dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        return pkv::fail(PKV_CUDA_ERROR, "cuTensorMapEncodeTiled (output) failed with code " + std::to_string(int(r)));
    }
    return PKV_OK;
}

int sm_count(int device) {
    static std::atomic<int> cached[kMaxDevices] = {};
    if (device >= 0 && device < kMaxDevices) {
        const int known = cached[device].load(std::memory_order_relaxed);
        if (known > 0) return known;
    }
    int sms = 148;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (device >= 0 && device < kMaxDevices && sms > 0) cached[device].store(sms, std::memory_order_relaxed);
    return sms;
}

// Raise a kernel's shared-memory limit once per device.
int prepare(const void *kernel, int smem, int device, std::atomic<int> *prepared) {
    const bool known = device >= 0 && device < kMaxDevices;
    if (known && prepared[device].load(std::memory_order_acquire)) return PKV_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
        return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 linear: cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    }
    if (known) prepared[device].store(1, std::memory_order_release);
    return PKV_OK;
}

template <typename... KernelArgs>
int launch_kernel(void (*kernel)(KernelArgs...), int grid, int threads, int smem, int cluster, cudaStream_t stream,
                  const KernelArgs &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 linear launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
}

int operand_maps(const void *x, int64_t x_stride, int x_box, const void *w, int w_box, int32_t k, const LinearArgs &args,
                 CUtensorMap *w_map, CUtensorMap *x_map) {
    const int rc = byte_matrix_map(w, static_cast<uint64_t>(args.n), static_cast<uint64_t>(k), static_cast<uint64_t>(k),
                                   static_cast<uint32_t>(w_box), w_map);
    if (rc) return rc;
    return byte_matrix_map(x, static_cast<uint64_t>(args.rows), static_cast<uint64_t>(k), static_cast<uint64_t>(x_stride),
                           static_cast<uint32_t>(x_box), x_map);
}

// CTAs that share a tile's K blocks: as many as still find a free slot, each keeping a block.
int row_splits(int64_t tiles, int k_blocks, int slots, int most) {
    int splits = 1;
    while (splits < most && tiles * splits * 2 <= slots && k_blocks >= 2 * splits) splits *= 2;
    return splits;
}

// Largest cluster of the kernel for many rows, which takes a whole SM a CTA: clusters of
// eight left SMs of a GPC idle and ran in two waves (128 x 2048 x 2048: 13.3 us, 8.0
// with four).
constexpr int kRowsCluster = 4;

template <int NT>
int launch_few(int device, const void *x, int64_t x_stride, const void *w, int32_t k, int sms, LinearArgs &args,
               cudaStream_t stream) {
    using S = Shape<NT>;
    static std::atomic<int> prepared[kMaxDevices] = {};
    int rc = prepare(reinterpret_cast<const void *>(fp8_linear_kernel<NT>), S::kSmem, device, prepared);
    if (rc) return rc;
    CUtensorMap w_map, x_map;
    if ((rc = operand_maps(x, x_stride, NT, w, kTileRows, k, args, &w_map, &x_map))) return rc;
    // Two CTAs fit an SM, which hides more of a K block's chain than long pieces save: at
    // 16 rows 11264 x 2048 takes 7.3 us (8.6 filling each SM once), 8192 x 2048 6.0 (6.8).
    args.splits = row_splits(args.n_tiles, args.k_blocks, 2 * sms, kMaxCluster);
    if (static_cast<int64_t>(args.n_tiles) * args.splits > INT32_MAX) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: too many tiles");
    }
    return launch_kernel(fp8_linear_kernel<NT>, args.n_tiles * args.splits, S::kThreads, S::kSmem, args.splits, stream,
                         w_map, x_map, args);
}

template <int N>
int launch_rows(int device, const void *x, int64_t x_stride, const void *w, int32_t k, int sms, LinearArgs &args,
                cudaStream_t stream) {
    using S = RowsShape<N>;
    static std::atomic<int> prepared[kMaxDevices] = {};
    int rc = prepare(reinterpret_cast<const void *>(fp8_linear_rows_kernel<N>), S::kSmem, device, prepared);
    if (rc) return rc;
    CUtensorMap w_map, x_map;
    if ((rc = operand_maps(x, x_stride, kTileRows, w, N, k, args, &w_map, &x_map))) return rc;
    const int64_t m_tiles = (static_cast<int64_t>(args.rows) + kTileRows - 1) / kTileRows;
    const int64_t tiles = m_tiles * ((static_cast<int64_t>(args.n) + N - 1) / N);
    if (tiles > INT32_MAX / kMaxCluster) return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: too many tiles");
    args.m_tiles = static_cast<int32_t>(m_tiles);
    args.tiles = static_cast<int32_t>(tiles);
    args.splits = row_splits(tiles, args.k_blocks, sms, kRowsCluster);
    const int64_t grid = args.splits > 1 ? tiles * args.splits : tiles < sms ? tiles : sms;
    return launch_kernel(fp8_linear_rows_kernel<N>, static_cast<int>(grid), S::kThreads, S::kSmem, args.splits, stream,
                         w_map, x_map, args);
}

// The pair kernel's warpgroups share out the registers it was planned to be launched with.
int check_registers(int device) {
    static std::atomic<int> checked[kMaxDevices] = {};
    const bool known = device >= 0 && device < kMaxDevices;
    if (known && checked[device].load(std::memory_order_acquire)) return PKV_OK;
    cudaFuncAttributes attributes;
    const cudaError_t e = cudaFuncGetAttributes(&attributes, reinterpret_cast<const void *>(fp8_linear_pair_kernel));
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 linear: cudaFuncGetAttributes: ") + cudaGetErrorString(e));
    if (attributes.numRegs < PairShape::kRegisters) {
        return pkv::fail(PKV_CUDA_ERROR, "fp8 linear: the pair kernel was compiled to fewer registers than its warps share out");
    }
    if (known) checked[device].store(1, std::memory_order_release);
    return PKV_OK;
}

int launch_pairs(int device, const void *x, int64_t x_stride, const void *w, int32_t k, int sms, LinearArgs &args,
                 cudaStream_t stream) {
    using S = PairShape;
    static std::atomic<int> prepared[kMaxDevices] = {};
    int rc = prepare(reinterpret_cast<const void *>(fp8_linear_pair_kernel), S::kSmem, device, prepared);
    if (rc) return rc;
    if ((rc = check_registers(device))) return rc;
    CUtensorMap w_map, x_map;
    if ((rc = operand_maps(x, x_stride, kTileRows, w, S::kN / 2, k, args, &w_map, &x_map))) return rc;
    const int64_t m_tiles = (static_cast<int64_t>(args.rows) + 255) / 256;
    const int64_t tiles = m_tiles * ((static_cast<int64_t>(args.n) + S::kN - 1) / S::kN);
    if (tiles > INT32_MAX / 2) return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: too many tiles");
    args.m_tiles = static_cast<int32_t>(m_tiles);
    args.tiles = static_cast<int32_t>(tiles);
    const int64_t pairs = tiles < sms / 2 ? tiles : sms / 2;
    CUtensorMap out_map = x_map;  // of no use to outputs that a tensor map cannot describe
    if (args.vector_out && (rc = half_matrix_map(args, 32, 32, &out_map))) return rc;
    return launch_kernel(fp8_linear_pair_kernel, static_cast<int>(2 * pairs), S::kThreads, S::kSmem, 2, stream, w_map, x_map,
                         out_map, args);
}

}  // namespace

extern "C" int pkv_fp8_linear(const void *x, int64_t x_stride, const void *x_scales, const void *w,
                              const void *w_scales, int32_t rows, int32_t n, int32_t k, void *out, int64_t out_stride,
                              int32_t *error_flag, void *stream) {
    pkv::clear_error();
    if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || out == nullptr ||
        error_flag == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: null pointer argument");
    }
    if (rows < 0 || n < 1 || k < 16 || k % 16) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: k must be a multiple of 16, n at least 1");
    }
    // A tile past the last row or column still counts in 32 bits.
    if (rows > INT32_MAX - 255 || n > INT32_MAX - 255 || k > INT32_MAX - 127) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: too many rows or columns");
    }
    if ((reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) || x_stride % 16 ||
        x_stride < k || (reinterpret_cast<uintptr_t>(out) & 1) || out_stride < n ||
        (reinterpret_cast<uintptr_t>(x_scales) & 3) || (reinterpret_cast<uintptr_t>(w_scales) & 3)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: misaligned tensor");
    }
    if (rows == 0) return PKV_OK;
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
    LinearArgs args;
    args.x_scales = static_cast<const float *>(x_scales);
    args.w_scales = static_cast<const float *>(w_scales);
    args.out = static_cast<__half *>(out);
    args.out_stride = out_stride;
    args.rows = rows;
    args.n = n;
    args.k_blocks = (k + kKBlock - 1) / kKBlock;
    args.splits = 1;
    args.n_tiles = (n + kTileRows - 1) / kTileRows;
    args.m_tiles = 0;
    args.tiles = 0;
    args.w_blocks = args.n_tiles;
    args.vector_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && out_stride % 8 == 0;
    args.error_flag = error_flag;
    const auto s = static_cast<cudaStream_t>(stream);
    const int sms = sm_count(device);
    if (rows <= 16) return launch_few<16>(device, x, x_stride, w, k, sms, args, s);
    if (rows <= 32) return launch_few<32>(device, x, x_stride, w, k, sms, args, s);
    if (rows <= 64) return launch_few<64>(device, x, x_stride, w, k, sms, args, s);
    // Tile shape by the time of the busiest SM: rounds of tiles, times the K blocks of a
    // CTA, times the clocks that a K block was measured to take: 700 / 800 / 1000 at
    // N = 64 / 128 / 192, and 1100 for a pair's 256 x 256.  Up to 192 that is mostly the
    // transfer of the block's 24 / 32 / 40 KiB from L2, 35 to 41 bytes a clock and SM: the
    // loads alone, without MMAs, TMEM reads and sums, take 9.4 of 12.0 us at 256 x 11264 x
    // 2048 (rows x n x k) and 15.6 of 20.5 at 512 rows.
    const int64_t m_tiles = (rows + kTileRows - 1) / kTileRows;
    const int64_t pair_rounds = (static_cast<int64_t>((rows + 255) / 256) * ((n + 255) / 256) + sms / 2 - 1) / (sms / 2);
    int best = 256;
    int64_t best_cost = pair_rounds * args.k_blocks * 1100;
    constexpr int kWidths[3] = {192, 128, 64}, kClocks[3] = {1000, 800, 700};
    for (int i = 0; i < 3; ++i) {
        const int64_t tiles = m_tiles * ((n + kWidths[i] - 1) / kWidths[i]);
        const int splits = row_splits(tiles, args.k_blocks, sms, kRowsCluster);
        const int64_t rounds = (tiles * splits + sms - 1) / sms;
        const int64_t cost = rounds * ((args.k_blocks + splits - 1) / splits) * kClocks[i];
        if (cost < best_cost) best = kWidths[i], best_cost = cost;
    }
    if (best == 256) return launch_pairs(device, x, x_stride, w, k, sms, args, s);
    if (best == 192) return launch_rows<192>(device, x, x_stride, w, k, sms, args, s);
    if (best == 128) return launch_rows<128>(device, x, x_stride, w, k, sms, args, s);
    return launch_rows<64>(device, x, x_stride, w, k, sms, args, s);
}
