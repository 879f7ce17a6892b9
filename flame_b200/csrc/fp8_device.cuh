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

struct Fp8Scale {
  float scale, inv;
  bool divide;
};

__device__ __forceinline__ Fp8Scale fp8_scale_of(float amax) {
  Fp8Scale s;
  s.scale = __fdiv_rn(amax, 448.0f);
  s.inv = s.scale == 0.0f ? 0.0f : __frcp_rn(s.scale);   // also where amax / 448 underflows to 0 (amax under 2^-141): codes of zero
  s.divide = s.inv > 3.0e38f;
  return s;
}

__device__ __forceinline__ float fp8_scaled(float x, const Fp8Scale& s) {
  if (s.divide) return __fdiv_rn(x, s.scale);
  return __fmul_rn(x, s.inv);
}

__device__ __forceinline__ uint32_t fp8_encode2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight elements of a block with absolute maximum amax.
__device__ __forceinline__ uint2 fp8_encode8(const float (&x)[8], const Fp8Scale& s) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = fp8_encode2(fp8_scaled(x[2 * i], s), fp8_scaled(x[2 * i + 1], s));
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
__device__ __forceinline__ uint2 fp8_encode8(const float (&x)[8], float amax, float& scale) {
  const Fp8Scale s = fp8_scale_of(amax);
  scale = s.scale;
  return fp8_encode8(x, s);
}

}  // namespace flame_b200
