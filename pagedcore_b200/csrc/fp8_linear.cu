// 8-bit linear layer on the sm_100a tensor cores:
//   y[m][n] = fp16( sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] * w[n][k] )
// with E4M3 codes x [rows][k] and w [n][k] and FP32 scales per row of x and
// 128 values, and per 128 x 128 block of w.
//
// The weight is the MMA's M side (128 weight rows a tile), the rows of x its N
// side (NT a tile, 16 to 256): at decode the weight is the large operand and is
// read once.  One K block of 128 is four tcgen05.mma (kind::f8f6f4, K = 32)
// into a TMEM buffer of its own; the scales differ from block to block, so a
// block's sums are read back and added into FP32 registers times sx * sw (sw is
// one number for the tile and block, sx one per column).  Two TMEM buffers let
// the tensor cores work on the next block meanwhile.
//
// Work split: one CTA per (128 weight rows, NT rows of x); where that leaves
// SMs idle the K blocks of a tile are dealt to the 2, 4 or 8 CTAs of a cluster,
// which add their FP32 sums through distributed shared memory in rank order and
// write FP16: one launch, and results that do not depend on timing.
//
// Roles: warps 0 .. E-1 read TMEM, scale and add (warp w reads lanes
// 32 (w % 4) .. and with E = 8 half of the columns); warp E loads by TMA (one
// 128-byte swizzled box of each operand a stage, no multicast); warp E + 1 owns
// the TMEM allocation and issues the MMAs.  Every wait is bounded; one that
// runs out sets PKV_DEVICE_WAIT_TIMEOUT, and the CTA goes on without waiting so
// that no barrier is left short.

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <functional>
#include <mutex>
#include <string>
#include <unordered_map>

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

template <int NT>
struct Shape {
    static constexpr int kEpilogueWarps = NT >= 128 ? 8 : 4;
    static constexpr int kThreads = (kEpilogueWarps + 2) * 32;
    static constexpr int kColumns = NT / (kEpilogueWarps / 4);  // of one epilogue warp
    static constexpr int kStageBytes = kWBytes + NT * kKBlock;
    static constexpr int kStages = NT >= 256 ? 4 : NT >= 128 ? 3 : 4;
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
    int32_t vector_out;  // rows of out take 8-byte stores
    int32_t *error_flag;
};

__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, int32_t *error_flag) {
    if (pkv::mbar_wait_bounded(bar, parity, kWaitPolls)) return true;
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
                 : "r"(addr)
                 : "memory");
    return v;
}

template <int NT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
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
    const int tile = static_cast<int>(blockIdx.x) / a.splits;
    const int n_tile = tile % a.n_tiles;
    const int n0 = n_tile * kTileRows;
    const int m0 = tile / a.n_tiles * NT;
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
            // The weight is no kernel's output: the first stages' weight boxes go out before the wait.
            const int early = min(count, S::kStages);
            for (int i = 0; i < early; ++i) {
                const uint32_t bar = pkv::smem_addr(&full[i]);
                pkv::mbar_arrive_expect_tx(bar, S::kStageBytes);
                pkv::tma_load_2d(base + i * S::kStageBytes, &w_map, (kb_begin + i) * kKBlock, n0, bar);
            }
            issued = early;
            pkv::pdl_wait();
            for (int i = 0; i < early; ++i) {
                pkv::tma_load_2d_hint(base + i * S::kStageBytes + kWBytes, &x_map, (kb_begin + i) * kKBlock, m0,
                                      pkv::smem_addr(&full[i]), reused);
            }
            for (int i = early; i < count; ++i) {
                const int st = i % S::kStages;
                if (!wait_bounded(pkv::smem_addr(&empty[st]), ((i / S::kStages) - 1) & 1, a.error_flag)) break;
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
        // Thread c < NT loads column c's scale, two K blocks ahead.
        const int column = m0 + static_cast<int>(threadIdx.x);
        const bool loads = threadIdx.x < NT;
        const bool inside = loads && column < a.rows;
        const float *sx = a.x_scales + static_cast<int64_t>(inside ? column : 0) * a.k_blocks + kb_begin;
        const float *sw = a.w_scales + static_cast<int64_t>(n_tile) * a.k_blocks + kb_begin;
        float f0 = inside ? sx[0] * sw[0] : 0.f;
        float f1 = inside && count > 1 ? sx[1] * sw[1] : 0.f;
        const int first = (warp >> 2) * S::kColumns;  // of this warp's columns
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        bool ok = true;
        for (int i = 0; i < count; ++i) {
            const int buf = i & 1;
            if (loads) factors[buf][threadIdx.x] = f0;
            f0 = f1;
            f1 = inside && i + 2 < count ? sx[i + 2] * sw[i + 2] : 0.f;
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
    // Rank r adds and writes columns r, r + splits, ...: a warp a column, four weight rows a lane.
    for (int c = split + a.splits * warp; c < NT && m0 + c < a.rows; c += a.splits * (S::kThreads / 32)) {
        const uint32_t at = static_cast<uint32_t>((c * kTileRows + 4 * lane) * 4);
        float4 v;
        if (a.splits == 1) {
            v = *reinterpret_cast<const float4 *>(reinterpret_cast<const uint8_t *>(sums) + at);
        } else {
            v = ld_cluster_f4(map_to_rank(base + at, 0));
            for (int s = 1; s < a.splits; ++s) {
                const float4 u = ld_cluster_f4(map_to_rank(base + at, s));
                v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            }
        }
        const int n = n0 + 4 * lane;
        __half *dst = a.out + static_cast<int64_t>(m0 + c) * a.out_stride + n;
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
// Host side.
// ---------------------------------------------------------------------------
constexpr int kMaxDevices = 64;

struct MapKey {
    uintptr_t base;
    uint64_t rows, cols, stride;
    uint32_t box_rows;
    bool operator==(const MapKey &o) const {
        return base == o.base && rows == o.rows && cols == o.cols && stride == o.stride && box_rows == o.box_rows;
    }
};
struct MapKeyHash {
    size_t operator()(const MapKey &k) const {
        return std::hash<uintptr_t>()(k.base) ^ (k.rows << 7) ^ (k.cols << 19) ^ (k.stride << 31) ^ k.box_rows;
    }
};

// A map holds an address and a shape only, so one that is found again is the one that would be made.
int byte_matrix_map(const void *base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t box_rows,
                    CUtensorMap *out) {
    static std::mutex mutex;
    static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
    const MapKey key{reinterpret_cast<uintptr_t>(base), rows, cols, stride, box_rows};
    std::lock_guard<std::mutex> lock(mutex);
    auto it = cache.find(key);
    if (it != cache.end()) {
        *out = it->second;
        return PKV_OK;
    }
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
    if (cache.size() > 4096) cache.clear();
    cache.emplace(key, *out);
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

template <int NT>
int launch(int device, const void *x, int64_t x_stride, const void *w, int32_t k, LinearArgs &args,
           cudaStream_t stream) {
    using S = Shape<NT>;
    static std::atomic<int> prepared[kMaxDevices] = {};
    if (device < 0 || device >= kMaxDevices || !prepared[device].load(std::memory_order_acquire)) {
        const cudaError_t e =
            cudaFuncSetAttribute(fp8_linear_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e != cudaSuccess) {
            return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 linear: cudaFuncSetAttribute: ") + cudaGetErrorString(e));
        }
        if (device >= 0 && device < kMaxDevices) prepared[device].store(1, std::memory_order_release);
    }
    CUtensorMap w_map, x_map;
    int rc = byte_matrix_map(w, static_cast<uint64_t>(args.n), static_cast<uint64_t>(k), static_cast<uint64_t>(k),
                             kTileRows, &w_map);
    if (rc) return rc;
    rc = byte_matrix_map(x, static_cast<uint64_t>(args.rows), static_cast<uint64_t>(k), static_cast<uint64_t>(x_stride),
                         NT, &x_map);
    if (rc) return rc;
    const int64_t tiles = static_cast<int64_t>(args.n_tiles) * ((args.rows + NT - 1) / NT);
    // Split K while the cluster's CTAs still find free SMs and each keeps a K block.
    int splits = 1;
    const int sms = sm_count(device);
    while (splits < kMaxCluster && tiles * splits * 2 <= sms + sms / 8 && args.k_blocks >= 2 * splits) splits *= 2;
    if (tiles * splits > INT32_MAX) return pkv::fail(PKV_VALUE_ERROR, "fp8 linear: too many tiles");
    args.splits = splits;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(tiles * splits));
    config.blockDim = dim3(S::kThreads);
    config.dynamicSmemBytes = S::kSmem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = static_cast<unsigned>(splits);
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = splits > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, fp8_linear_kernel<NT>, w_map, x_map, args);
    if (e != cudaSuccess) return pkv::fail(PKV_CUDA_ERROR, std::string("fp8 linear launch failed: ") + cudaGetErrorString(e));
    return PKV_OK;
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
    args.vector_out = (reinterpret_cast<uintptr_t>(out) & 7) == 0 && out_stride % 4 == 0;
    args.error_flag = error_flag;
    const auto s = static_cast<cudaStream_t>(stream);
    if (rows <= 16) return launch<16>(device, x, x_stride, w, k, args, s);
    if (rows <= 32) return launch<32>(device, x, x_stride, w, k, args, s);
    if (rows <= 64) return launch<64>(device, x, x_stride, w, k, args, s);
    if (rows <= 128) return launch<128>(device, x, x_stride, w, k, args, s);
    return launch<256>(device, x, x_stride, w, k, args, s);
}
