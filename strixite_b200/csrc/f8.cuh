// Codes of 8-bit floating point (e4m3) with an FP32 scale for every block of 128 along a row: element = code * scale.  What the kernels that make
// and read them share.
#pragma once

#include "common.cuh"

namespace sxb {

constexpr int kF8Block = 128;
constexpr float kF8Top = 448.0f;        // the largest e4m3 number
constexpr float kF8Least = 0x1p-64f;    // of a scale: its reciprocal stays a normal FP32 number, and its product with another scale loses no more than 2^-22 (2^-128 and more: the least ones are subnormal)

// The scale of a block, `exact` the 448th part of its largest magnitude: NaN if that is NaN or beyond FP32.
__device__ inline float f8_scale(float exact) { return exact < INFINITY ? fmaxf(exact, kF8Least) : qnan_f32(); }
__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Two values to two codes (the first in the lower byte): nearest, ties to even, beyond +-448 the last number, NaN stays NaN.
__device__ inline uint32_t f8_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ inline uint32_t f8_quad(float a, float b, float c, float d) { return f8_pair(a, b) | (f8_pair(c, d) << 16); }

// Two values rounded to BF16 (the first in the lower half).
__device__ inline uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace sxb
