// Dropout from a counter-based generator, written for sm_100a: the mask is a function of (seed, offset, element index) and is
// never stored.  The backward pass, and a forward pass that is run again under gradient checkpointing, compute it again.
//
// Generator: Philox 4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", SC11).  One call gives 128 bits, which serve the eight elements of a group as eight 16-bit numbers; with p = t / 2^32 an
// element is dropped when its 32-bit number is under t.  The 16 bits decide unless they equal t's upper half, which happens once
// in 65,536 elements: only then are the lower 16 bits drawn, from the counter with bit 63 set.  So the probability is exact to
// 2^-32 at the price of 16 bits per element.
//
//   group g = i / 8, counter (g mod 2^32, g / 2^32, offset mod 2^32, offset / 2^32), key = (seed mod 2^32, seed / 2^32);
//   u(i) = half(i mod 8) of philox(counter) * 2^16 + half(i mod 8) of philox(counter with bit 63 of g set)
//   y[i] = u(i) >= t ? x[i] / (1 - p) : 0, plus residual[i] where there is one; fp32 inside, rounded once.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "codec_kernels.cuh"
#include "common.h"

namespace flame_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;

struct DropoutArgs {
  const void* x;
  const void* residual;          // may be NULL
  void* y;
  size_t n;
  const uint64_t* seed_device;   // NULL: `seed` is used
  uint64_t seed, offset;
  uint32_t t_hi, t_lo;           // t_hi = 65536 drops everything
  float scale;
};

__device__ __forceinline__ uint4 philox10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// bit j: element j of the group is kept
__device__ __forceinline__ uint32_t keep_bits(uint64_t g, const DropoutArgs& a, uint64_t seed) {
  const uint32_t lo = (uint32_t)g, hi = (uint32_t)(g >> 32), o0 = (uint32_t)a.offset, o1 = (uint32_t)(a.offset >> 32);
  const uint4 w = philox10(lo, hi, o0, o1, (uint32_t)seed, (uint32_t)(seed >> 32));
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
  uint32_t keep = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    const uint32_t h = (j & 1) ? ws[j / 2] >> 16 : ws[j / 2] & 0xFFFFu;
    keep |= (h >= a.t_hi) ? 1u << j : 0u;
    tie |= (h == a.t_hi) ? 1u << j : 0u;
  }
  if (tie != 0 && a.t_lo != 0) {
    const uint4 v = philox10(lo, hi | 0x80000000u, o0, o1, (uint32_t)seed, (uint32_t)(seed >> 32));
    const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      const uint32_t h = (j & 1) ? vs[j / 2] >> 16 : vs[j / 2] & 0xFFFFu;
      if (((tie >> j) & 1u) && h < a.t_lo) keep &= ~(1u << j);
    }
  }
  return keep;
}

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }

template <typename T>
struct alignas(16) Group { T v[kGroup]; };   // 16 bytes of BF16, 32 of binary32

// kVec: whole groups move as 16-byte accesses (16-byte aligned tensors).  The last, shorter group goes element by element.
template <typename T, bool kVec, bool kResidual>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ DropoutArgs a) {
  pdl_prologue();
  const uint64_t seed = a.seed_device ? *a.seed_device : a.seed;
  const size_t groups = (a.n + kGroup - 1) / kGroup;
  const T* __restrict__ x = static_cast<const T*>(a.x);
  const T* __restrict__ res = static_cast<const T*>(a.residual);
  T* __restrict__ y = static_cast<T*>(a.y);
  for (size_t g = (size_t)blockIdx.x * kThreads + threadIdx.x; g < groups; g += (size_t)gridDim.x * kThreads) {
    const size_t i0 = g * kGroup;
    const int count = a.n - i0 < kGroup ? (int)(a.n - i0) : kGroup;
    Group<T> xv, rv, yv;
    const bool whole = kVec && count == kGroup;
    if (whole) {
      xv = *reinterpret_cast<const Group<T>*>(x + i0);
      if (kResidual) rv = *reinterpret_cast<const Group<T>*>(res + i0);
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        if (j < count) { xv.v[j] = x[i0 + j]; if (kResidual) rv.v[j] = res[i0 + j]; }
    }
    const uint32_t keep = keep_bits(g, a, seed);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      // selected, not multiplied by 0: a dropped infinity or NaN leaves nothing behind
      float v = ((keep >> j) & 1u) ? __fmul_rn(to_f(xv.v[j]), a.scale) : 0.0f;
      if (kResidual) v = __fadd_rn(to_f(rv.v[j]), v);
      from_f(yv.v[j], v);
    }
    if (whole) {
      *reinterpret_cast<Group<T>*>(y + i0) = yv;
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        if (j < count) y[i0 + j] = yv.v[j];
    }
  }
}

template <typename T>
cudaError_t launch_dropout_t(const DropoutArgs& a, cudaStream_t stream) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool vec = al(a.x) && al(a.y) && al(a.residual);
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const size_t blocks = ((a.n + kGroup - 1) / kGroup + kThreads - 1) / kThreads;
  const size_t cap = (size_t)sms * 8 * 4;
  const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
  auto go = [&](auto kern) { return launch_after(kern, grid, kThreads, 0, stream, a); };
  if (a.residual) return vec ? go(dropout_kernel<T, true, true>) : go(dropout_kernel<T, false, true>);
  return vec ? go(dropout_kernel<T, true, false>) : go(dropout_kernel<T, false, false>);
}

}  // namespace
}  // namespace flame_b200

using namespace flame_b200;

extern "C" int flame_dropout(const void* x, const void* residual, void* y, size_t n, int dtype, double p, uint64_t seed,
                             const void* seed_device, uint64_t offset, void* stream) {
  if (!(p >= 0.0 && p <= 1.0)) {
    set_last_error("flame_dropout: p must be in [0, 1]");
    return (int)cudaErrorInvalidValue;
  }
  if (dtype != FLAME_OFFLOAD_DTYPE_BF16 && dtype != FLAME_OFFLOAD_DTYPE_F32) {
    set_last_error("flame_dropout: dtype must be BF16 or F32");
    return (int)cudaErrorInvalidValue;
  }
  if (n == 0) return 0;
  if (!x || !y) {
    set_last_error("flame_dropout: null tensor");
    return (int)cudaErrorInvalidValue;
  }
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return (int)cudaErrorLaunchFailure;
  const double t = nearbyint(p * 4294967296.0);   // 0 .. 2^32
  const uint64_t ti = (uint64_t)t;
  DropoutArgs a;
  a.x = x; a.residual = residual; a.y = y; a.n = n;
  a.seed_device = static_cast<const uint64_t*>(seed_device);
  a.seed = seed; a.offset = offset;
  a.t_hi = (uint32_t)(ti >> 16); a.t_lo = (uint32_t)(ti & 0xFFFFu);
  a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  return dtype == FLAME_OFFLOAD_DTYPE_BF16 ? (int)launch_dropout_t<__nv_bfloat16>(a, (cudaStream_t)stream)
                                           : (int)launch_dropout_t<float>(a, (cudaStream_t)stream);
}
