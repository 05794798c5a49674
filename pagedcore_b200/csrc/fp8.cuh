// E4M3 values with power-of-two scales: the 8-bit form shared by the 8-bit
// rows (activations) and the 8-bit KV cache.
//
// A block of values is stored as codes and one FP32 scale s = 2^e, the value
// of a code c being c * s.  e is the smallest exponent in [-15, 8] for which
// the block's largest magnitude is at most 448 s.  Why a power of two: E4M3 is
// a floating format, so a scale that uses up the last fraction of an octave
// gains no precision, while with a power of two the division, the product and
// a later change of scale are exact (a raised scale only moves codes into the
// subnormals), and every value is an FP16 number: at e = -15 the smallest
// step is 2^-9 * 2^-15 = 2^-24, FP16's own, and at e = 8 codes stop at 240
// (240 * 256 = 61440 <= 65504).  Rounding: to nearest, ties to even, half a
// step or 2^-4 of the value.  A value that is not finite is stored as NaN and
// takes no part in the scale.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace pkv::fp8 {

constexpr int kMinExponent = -15;
constexpr int kMaxExponent = 8;
constexpr int kGroup = 128;  // values per scale of 8-bit rows

// max(|x|, m), x left out when it is not finite.
__device__ __forceinline__ float max_finite(float m, float x) {
    const float a = fabsf(x);
    return a < __int_as_float(0x7f800000) ? fmaxf(m, a) : m;
}

// Exponent of the scale of a block with the largest magnitude `amax` (finite,
// >= 0): 448 = 1.75 * 2^8, so amax = f * 2^x needs x - 8, and one more where f
// is above 1.75 (fraction bits above 0x600000: the sum carries).
__device__ __forceinline__ int scale_exponent(float amax) {
    const int e = ((__float_as_int(amax) + 0x1fffff) >> 23) - 127 - 8;
    return min(max(e, kMinExponent), kMaxExponent);
}

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of a stored scale; held within the range so that a scale that was
// never written cannot make another one.
__device__ __forceinline__ int stored_exponent(float scale) {
    const int e = ((__float_as_int(scale) >> 23) & 0xff) - 127;
    return min(max(e, kMinExponent), kMaxExponent);
}

// x as the conversion takes it: times 2^-e, not finite -> NaN, and at the
// largest scale at most 240 (so that the value stays an FP16 number).
__device__ __forceinline__ float scaled(float x, float inverse, bool largest) {
    const float v = fmaf(x, 0.f, x) * inverse;  // inf * 0 is NaN
    return largest && fabsf(v) > 240.f ? copysignf(240.f, v) : v;
}

// Two values to codes (lo in the low byte), rounded to nearest even, NaN kept.
__device__ __forceinline__ uint32_t encode2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two codes (low 16 bits of `codes`) to the FP16 numbers they stand for.
__device__ __forceinline__ uint32_t decode2(uint32_t codes) {
    uint32_t r;
    const uint16_t c = static_cast<uint16_t>(codes);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}

// Four codes to two such pairs (the halves of a register are operands of their own: no shift).
__device__ __forceinline__ void decode4(uint32_t codes, uint32_t &low, uint32_t &high) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(low), "=r"(high)
        : "r"(codes));
}

__device__ __forceinline__ float2 decode2f(uint32_t codes) {
    const uint32_t h = decode2(codes);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Codes moved to a scale 2^-shift times as fine, i.e. code * factor with
// factor = 2^(e_old - e_new) < 1, four at a time.
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float factor) {
    const float2 a = decode2f(codes), b = decode2f(codes >> 16);
    return encode2(a.x * factor, a.y * factor) | (encode2(b.x * factor, b.y * factor) << 16);
}

}  // namespace pkv::fp8
