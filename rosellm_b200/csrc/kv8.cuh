// The 8-bit cache: its number format and what its kernels share.
//
// A cached value is code * scale: an e4m3 code (float8_e4m3fn: four exponent bits, three of fraction, no infinity, largest
// 448) and the float32 scale of its block.  A block is 16 consecutive tokens of one page, one plane (keys or values) and one
// key/value head; its scale is the smallest power of two s >= 2^-126 with |x| <= 448 s for all that was written into it.  Powers of two,
// because dividing by them is exact: a value is rounded once, to its code (half a step, 2^-4 relative, above 2^-6 s), and when a later
// token raises its block's scale the codes of the earlier ones move by whole exponents, which is exact but for those that
// fall below 2^-6 of the new scale.
//
// Layout of one layer: codes [pages][2][kv heads][page size][head dim], scales [pages][2][kv heads][page size / 16].
#pragma once
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace rl {
namespace kv8 {

constexpr int BLOCK = 16;  // tokens that share a scale; also the inner size of one mma.sync, so a step of P V has one scale

// The smallest power of two s >= 2^-126 with a <= 448 s, for finite a >= 0.  a = m 2^e with 1 <= m < 2 and 448 = 1.75 * 2^8: 2^(e-8) where
// m <= 1.75, else twice that.
__device__ __forceinline__ float scale_for(float a) {
  const uint32_t bits = __float_as_uint(a);
  int e = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);  // (subnormal a: e is negative)
}

// 1 / s for a power of two from 2^-126 to 2^126.
__device__ __forceinline__ float inverse_of(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// Two floats to two codes, nearest, ties to even; `lo` in the low byte.  NaN stays NaN; an infinity would become 448, and is turned into NaN before.
__device__ __forceinline__ uint16_t encode2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two codes to two halves (exact: every code is a half).
__device__ __forceinline__ uint32_t decode2(uint16_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
  return r;
}

}  // namespace kv8
}  // namespace rl
