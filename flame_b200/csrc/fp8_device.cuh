// FP8 E4M3 codes with one fp32 scale for a block of 128 elements, as the product's operands: the definitions that the quantiser
// and the group norm share.
//
//   scale = RN(absmax / 448); code = e4m3(RN(x * RN(1 / scale))), round to nearest even, saturating (the OCP encoder,
//   FLAME_ACT_FP8_OCP).  absmax ignores NaN; a NaN element gets a NaN code whatever its block, so that a product shows it.
//   A block without a value other than zero has scale 0 and codes of zero.  Where 1 / scale overflows (scale under 2^-128) the
//   elements are divided by the scale.  A block with an infinity has an infinite scale: its infinities become NaN codes.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace flame_b200 {

// max(|a|, |b|) of two packed BF16 pairs in one instruction; the sign bits of the result mean nothing.  A NaN operand is ignored.
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The larger of a packed pair of magnitudes as a binary32 number; NaN counts as zero.
__device__ __forceinline__ float larger_of(uint32_t pair) {
  return fmaxf(fmaxf(__uint_as_float((pair << 16) & 0x7FFF0000u), __uint_as_float(pair & 0x7FFF0000u)), 0.0f);
}

__device__ __forceinline__ float fp8_scale_of(float amax) { return __fdiv_rn(amax, 448.0f); }
// The factor of the elements.  Infinite where they have to be divided by the scale; 0 for a scale of 0 (also where amax / 448
// underflows, amax under 2^-141).
__device__ __forceinline__ float fp8_factor_of(float scale) { return scale == 0.0f ? 0.0f : __frcp_rn(scale); }
__device__ __forceinline__ bool fp8_divides(float factor) { return factor > 3.0e38f; }

__device__ __forceinline__ uint32_t fp8_encode2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 fp8_pack8(const float (&y)[8]) {
  return make_uint2(fp8_encode2(y[0], y[1]) | (fp8_encode2(y[2], y[3]) << 16), fp8_encode2(y[4], y[5]) | (fp8_encode2(y[6], y[7]) << 16));
}
// Two elements times their factors, one multiplication for both.
__device__ __forceinline__ uint64_t fp8_factors(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint32_t fp8_encode2(float lo, float hi, uint64_t factors) {
  uint16_t r;
  asm("{ .reg .b64 v; .reg .f32 a, b; mov.b64 v, {%1, %2}; mul.rn.f32x2 v, v, %3; mov.b64 {a, b}, v; cvt.rn.satfinite.e4m3x2.f32 %0, b, a; }"
      : "=h"(r) : "f"(lo), "f"(hi), "l"(factors));
  return r;
}
// Eight elements of one block.
__device__ __forceinline__ uint2 fp8_encode8(const float (&x)[8], float scale, float factor) {
  float y[8];
  if (fp8_divides(factor)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(x[i], scale);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(x[i], factor);
  }
  return fp8_pack8(y);
}
__device__ __forceinline__ void unpack8(const uint4& raw, float (&f)[8]) {   // eight BF16 numbers
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}

}  // namespace flame_b200
