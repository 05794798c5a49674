// 8-bit rows: E4M3 codes [rows][width] with one scale per row and 128 values
// (the last group may be shorter), the left operand of the 8-bit linear layer.
//
//   pkv_fp8_add_rms_norm  v = hidden + delta;  residual = fp16(v);
//                         y = v * rsqrt(mean(v^2) + eps) * weight
//   pkv_fp8_quantize      y = x, or with silu_pairs y = silu(gate) * up
// each computed in FP32 from FP16 inputs and rounded once, to E4M3.  (The FP16
// norm and SwiGLU round at every step of the eager chain they replace;
// here the 8-bit rounding is the only one.)  pkv_fp8_to_half gives the FP16
// numbers that 8-bit rows stand for, which are exact.
//
// Bound by launch latency to a few hundred rows (1.1 to 3.5 us at 1 and 256), above by
// memory in part: 2047 rows of 2048 take 6.2 us in the norm (bytes at the copy rate 4.5),
// 3.9 as plain rows (1.9), of 2 x 5632 17.7 in SwiGLU (8.8).
// Sixteen neighbouring lanes hold the 128 values of a group, eight each (one
// 16-byte load), so the group's maximum is four butterfly steps and the codes
// leave as one 8-byte store a lane.

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "fp8.cuh"
#include "pagedkv.h"
#include "pdl.h"
#include "ptx.cuh"
#include "status.h"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8;  // FP16 values per 16-byte access
constexpr int kMaxChunks = 4;
constexpr int kMaxDim = kThreads * kChunk * kMaxChunks;  // 8192
constexpr int kMaxRows = INT32_MAX - 65535;  // the row loops step by up to 65535 rows past the last

__device__ __forceinline__ void unpack8(const uint4 &raw, float (&v)[kChunk]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// The codes of a lane's eight values and the scale of the group that it shares
// with the 15 other lanes of its half warp (all 32 lanes call this).
__device__ __forceinline__ uint2 encode_group(const float (&y)[kChunk], float &scale) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) amax = pkv::fp8::max_finite(amax, y[i]);
#pragma unroll
    for (int offset = 8; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, offset));
    const int e = pkv::fp8::scale_exponent(amax);
    const bool largest = e == pkv::fp8::kMaxExponent;
    const float inverse = pkv::fp8::exp2_int(-e);
    scale = pkv::fp8::exp2_int(e);
    float s[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) s[i] = pkv::fp8::scaled(y[i], inverse, largest);
    return make_uint2(pkv::fp8::encode2(s[0], s[1]) | (pkv::fp8::encode2(s[2], s[3]) << 16),
                      pkv::fp8::encode2(s[4], s[5]) | (pkv::fp8::encode2(s[6], s[7]) << 16));
}

// (No __restrict__ on the inputs below: it promises that they do not change while the kernel
// runs, but a kernel launched early runs beside the one that writes them, and the norm's
// residual may be hidden or delta itself.  A thread reads all of its row before it writes.)

// One CTA per row; thread c holds chunk c (+ 256 ...) of the row.
template <int CHUNKS>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __half *hidden, const __half *delta, const __half *weight,
                                                        __half *residual, uint8_t *codes, float *scales, int dim,
                                                        int groups, float eps) {
    __shared__ float partial[kThreads / 32];
    const int chunks = dim / kChunk;
    uint4 wraw[CHUNKS], hraw[CHUNKS], draw[CHUNKS];
    pkv::pdl_launch_dependents();
    pkv::pdl_wait();
    const int64_t base = static_cast<int64_t>(blockIdx.x) * dim;
    float v[CHUNKS][kChunk];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = threadIdx.x + j * kThreads;
        wraw[j] = hraw[j] = draw[j] = make_uint4(0, 0, 0, 0);
        if (c < chunks) {
            wraw[j] = *reinterpret_cast<const uint4 *>(weight + c * kChunk);
            hraw[j] = *reinterpret_cast<const uint4 *>(hidden + base + c * kChunk);
            if (delta != nullptr) draw[j] = *reinterpret_cast<const uint4 *>(delta + base + c * kChunk);
        }
    }
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = threadIdx.x + j * kThreads;
        if (c < chunks) {
            unpack8(hraw[j], v[j]);
            if (delta != nullptr) {
                float d[kChunk];
                unpack8(draw[j], d);
                uint4 rraw;
                __half2 *r = reinterpret_cast<__half2 *>(&rraw);
#pragma unroll
                for (int i = 0; i < kChunk; ++i) v[j][i] += d[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = __floats2half2_rn(v[j][2 * i], v[j][2 * i + 1]);
                *reinterpret_cast<uint4 *>(residual + base + c * kChunk) = rraw;
            }
#pragma unroll
            for (int i = 0; i < kChunk; ++i) sum += v[j][i] * v[j][i];
        } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[j][i] = 0.f;
        }
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = sum;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) total += partial[w];
    const float inv = rsqrtf(total / static_cast<float>(dim) + eps);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = threadIdx.x + j * kThreads;
        float w[kChunk], y[kChunk], scale;
        unpack8(wraw[j], w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) y[i] = v[j][i] * inv * w[i];
        const uint2 out = encode_group(y, scale);
        if (c < chunks) {
            *reinterpret_cast<uint2 *>(codes + base + c * kChunk) = out;
            if ((threadIdx.x & 15) == 0) {
                scales[static_cast<int64_t>(blockIdx.x) * groups + c / (pkv::fp8::kGroup / kChunk)] = scale;
            }
        }
    }
}

// y = x, or with SILU y = silu(x[.., c]) * x[.., width + c]: 16 lanes a group,
// groups of a row along x, rows along y.
template <bool SILU>
__global__ void __launch_bounds__(kThreads) encode_kernel(const __half *x, int64_t stride, int rows, int width,
                                                          int groups, uint8_t *codes, float *scales) {
    pkv::pdl_launch_dependents();
    pkv::pdl_wait();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    const bool inside = c * kChunk < width;
    for (int row = blockIdx.y; row < rows; row += gridDim.y) {
        float y[kChunk];
        if (inside) {
            const __half *src = x + row * stride + c * kChunk;
            unpack8(*reinterpret_cast<const uint4 *>(src), y);
            if (SILU) {
                float u[kChunk];
                unpack8(*reinterpret_cast<const uint4 *>(src + width), u);
#pragma unroll
                for (int i = 0; i < kChunk; ++i) y[i] = y[i] / (1.0f + expf(-y[i])) * u[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) y[i] = 0.f;
        }
        float scale;
        const uint2 out = encode_group(y, scale);
        if (inside) {
            *reinterpret_cast<uint2 *>(codes + static_cast<int64_t>(row) * width + c * kChunk) = out;
            if ((threadIdx.x & 15) == 0) {
                scales[static_cast<int64_t>(row) * groups + c / (pkv::fp8::kGroup / kChunk)] = scale;
            }
        }
    }
}

__global__ void __launch_bounds__(kThreads) to_half_kernel(const uint8_t *codes, const float *scales, int rows,
                                                           int width, int groups, __half *out, int64_t out_stride) {
    pkv::pdl_launch_dependents();
    pkv::pdl_wait();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c * kChunk >= width) return;
    for (int row = blockIdx.y; row < rows; row += gridDim.y) {
        const uint2 in = *reinterpret_cast<const uint2 *>(codes + static_cast<int64_t>(row) * width + c * kChunk);
        const float s = scales[static_cast<int64_t>(row) * groups + c / (pkv::fp8::kGroup / kChunk)];
        uint4 raw;
        __half2 *h = reinterpret_cast<__half2 *>(&raw);
        const uint32_t words[2] = {in.x, in.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = pkv::fp8::decode2f(words[i >> 1] >> (16 * (i & 1)));
            h[i] = __floats2half2_rn(f.x * s, f.y * s);
        }
        *reinterpret_cast<uint4 *>(out + row * out_stride + c * kChunk) = raw;
    }
}

bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int groups_of(int width) { return (width + pkv::fp8::kGroup - 1) / pkv::fp8::kGroup; }

dim3 row_grid(int rows, int width) {
    return dim3((width / kChunk + kThreads - 1) / kThreads, static_cast<unsigned>(rows < 65535 ? rows : 65535));
}

int launched(cudaError_t err, const char *what) {
    if (err == cudaSuccess) return PKV_OK;
    return pkv::fail(PKV_CUDA_ERROR, std::string(what) + " launch failed: " + cudaGetErrorString(err));
}

}  // namespace

extern "C" int pkv_fp8_add_rms_norm(const void *hidden, const void *delta, const void *weight, void *residual,
                                    void *codes, void *scales, int32_t rows, int32_t dim, float eps, void *stream) {
    pkv::clear_error();
    if (hidden == nullptr || weight == nullptr || codes == nullptr || scales == nullptr ||
        (delta != nullptr && residual == nullptr)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rms norm: hidden, weight, codes and scales are required, and residual with delta");
    }
    if (rows > kMaxRows) return pkv::fail(PKV_VALUE_ERROR, "fp8 rms norm: too many rows");
    if (rows < 0 || dim < kChunk || dim % kChunk || dim > kMaxDim) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rms norm: dim must be a multiple of 8 up to 8192");
    }
    if (!aligned(hidden, 16) || !aligned(weight, 16) || !aligned(codes, 8) || !aligned(scales, 4) ||
        (delta && (!aligned(delta, 16) || !aligned(residual, 16)))) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rms norm: tensors must be 16-byte aligned (codes 8)");
    }
    if (rows == 0) return PKV_OK;
    const int per_thread = (dim / kChunk + kThreads - 1) / kThreads;
    const auto kernel = per_thread == 1 ? norm_kernel<1> : per_thread == 2 ? norm_kernel<2> : norm_kernel<4>;
    return launched(pkv::launch_pdl(kernel, dim3(rows), dim3(kThreads), static_cast<cudaStream_t>(stream),
                                    static_cast<const __half *>(hidden), static_cast<const __half *>(delta),
                                    static_cast<const __half *>(weight), static_cast<__half *>(residual),
                                    static_cast<uint8_t *>(codes), static_cast<float *>(scales), dim, groups_of(dim),
                                    eps),
                    "fp8 rms norm");
}

extern "C" int pkv_fp8_quantize(const void *x, int64_t x_stride, int32_t silu_pairs, int32_t rows, int32_t width,
                                void *codes, void *scales, void *stream) {
    pkv::clear_error();
    if (x == nullptr || codes == nullptr || scales == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: x, codes and scales are required");
    }
    if (rows > kMaxRows) return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: too many rows");
    if (rows < 0 || width < kChunk || width % kChunk || width > (1 << 28)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: the width must be a multiple of 8");
    }
    if (!aligned(x, 16) || !aligned(codes, 8) || !aligned(scales, 4) || x_stride % kChunk ||
        x_stride < static_cast<int64_t>(width) * (silu_pairs ? 2 : 1)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: x must be 16-byte aligned with a row stride in multiples of 8");
    }
    if (rows == 0) return PKV_OK;
    return launched(pkv::launch_pdl(silu_pairs ? encode_kernel<true> : encode_kernel<false>, row_grid(rows, width),
                                    dim3(kThreads), static_cast<cudaStream_t>(stream), static_cast<const __half *>(x),
                                    x_stride, rows, width, groups_of(width), static_cast<uint8_t *>(codes),
                                    static_cast<float *>(scales)),
                    "fp8 rows");
}

extern "C" int pkv_fp8_to_half(const void *codes, const void *scales, int32_t rows, int32_t width, void *out,
                               int64_t out_stride, void *stream) {
    pkv::clear_error();
    if (out == nullptr || codes == nullptr || scales == nullptr) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: codes, scales and out are required");
    }
    if (rows > kMaxRows) return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: too many rows");
    if (rows < 0 || width < kChunk || width % kChunk || width > (1 << 28)) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: the width must be a multiple of 8");
    }
    if (!aligned(out, 16) || !aligned(codes, 8) || !aligned(scales, 4) || out_stride % kChunk || out_stride < width) {
        return pkv::fail(PKV_VALUE_ERROR, "fp8 rows: out must be 16-byte aligned with a row stride in multiples of 8");
    }
    if (rows == 0) return PKV_OK;
    return launched(pkv::launch_pdl(to_half_kernel, row_grid(rows, width), dim3(kThreads),
                                    static_cast<cudaStream_t>(stream), static_cast<const uint8_t *>(codes),
                                    static_cast<const float *>(scales), rows, width, groups_of(width),
                                    static_cast<__half *>(out), out_stride),
                    "fp8 rows");
}
