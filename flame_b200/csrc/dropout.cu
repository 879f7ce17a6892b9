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

#include <type_traits>

#include "codec_kernels.cuh"
#include "common.h"

namespace flame_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;

// The generator's keys of its ten rounds.  From the host's seed they are constants of the launch; from a seed in device memory every
// thread makes them.
struct Keys { uint32_t k0[10], k1[10]; };
__host__ __device__ __forceinline__ void make_keys(uint64_t seed, Keys& k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) { k.k0[r] = (uint32_t)seed + r * 0x9E3779B9u; k.k1[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u; }
}

struct DropoutArgs {
  const void* x;
  const void* residual;          // may be NULL
  void* y;
  size_t n;
  const uint64_t* seed_device;   // NULL: `keys` are used
  Keys keys;
  uint32_t o0, o1;               // the offset's halves
  uint32_t t_hi, t_lo;           // the threshold's halves
  float scale;
};

__device__ __forceinline__ uint4 philox10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, const Keys& k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k.k0[r];
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k.k1[r];
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}

// keep[j]: element j of group g is kept.  The upper half of a word is compared where it is, the lower half shifted up.
__device__ __forceinline__ void kept(uint64_t g, const DropoutArgs& a, const Keys& k, bool (&keep)[kGroup]) {
  const uint4 w = philox10((uint32_t)g, (uint32_t)(g >> 32), a.o0, a.o1, k);
  const uint32_t t = a.t_hi << 16;
  const uint32_t h[kGroup] = {w.x << 16, w.x, w.y << 16, w.y, w.z << 16, w.z, w.w << 16, w.w};
  bool tie = false;
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    keep[j] = h[j] >= t;
    tie |= h[j] - t < 65536u;      // the upper 16 bits are the threshold's
  }
  if (tie && a.t_lo != 0) {
    const uint4 v = philox10((uint32_t)g, (uint32_t)(g >> 32) | 0x80000000u, a.o0, a.o1, k);
    const uint32_t l[kGroup] = {v.x & 0xFFFFu, v.x >> 16, v.y & 0xFFFFu, v.y >> 16, v.z & 0xFFFFu, v.z >> 16, v.w & 0xFFFFu, v.w >> 16};
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (h[j] - t < 65536u && l[j] < a.t_lo) keep[j] = false;
  }
}

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }

// A group in 16-byte pieces: one of BF16, two of binary32.
template <typename T>
constexpr int kPieces = kGroup * (int)sizeof(T) / 16;
template <typename T>
__device__ __forceinline__ void unpack(const uint4 (&r)[kPieces<T>], float (&f)[kGroup]) {
#pragma unroll
  for (int k = 0; k < kPieces<T>; ++k) {
    const uint32_t w[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
      else f[4 * k + i] = __uint_as_float(w[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store(T* p, const float (&f)[kGroup]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) reinterpret_cast<float4*>(p)[k] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
  }
}
// What is added to an element's residual, rounded once with it.  A dropped element is selected away, not multiplied by 0: an infinity or
// NaN leaves nothing behind.
__device__ __forceinline__ float value(bool keep, float x, float scale) { return keep ? __fmul_rn(x, scale) : 0.0f; }

// Whole groups of 16-byte aligned tensors.  The groups ahead are on their way to shared memory as asynchronous copies, each thread's
// own in places of its own: with one group in flight a thread (in registers) a 9216 x 9216 BF16 tensor took 94 us, the warps waiting
// for memory four cycles of ten.  Some 20 issue slots an element, half of them the generator's, where the copy rate of BF16 leaves 21:
// bound by both.  9216 x 9216 on one B200: BF16 71.5 us (4.7 TB/s), with a residual 78.7 us (6.5 TB/s), F32 108 us (6.3 TB/s), with a
// residual 152 us (6.7 TB/s), recorded in a CUDA graph and replayed back to back.
constexpr int kRingBytes = 32 * 1024;
template <typename T, bool kResidual, bool kDeviceSeed>
__global__ void __launch_bounds__(kThreads, 4) dropout_kernel(const __grid_constant__ DropoutArgs a) {
  pdl_prologue();
  constexpr int kP = kPieces<T>, kN = kResidual ? 2 : 1, kD = kRingBytes / (kThreads * 16 * kP * kN);
  __shared__ uint4 ring[kD * kN * kP * kThreads];
  Keys made;
  if (kDeviceSeed) make_keys(*a.seed_device, made);
  const Keys& keys = kDeviceSeed ? made : a.keys;
  const size_t groups = a.n / kGroup, turn = (size_t)gridDim.x * kThreads;
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(ring + threadIdx.x);
  size_t next = (size_t)blockIdx.x * kThreads + threadIdx.x;
  auto send = [&](int j) {
    if (next < groups) {
#pragma unroll
      for (int k = 0; k < kN * kP; ++k) {
        const uint32_t dst = at + (j * kN * kP + k) * kThreads * 16;
        const uint4* src = static_cast<const uint4*>(k < kP ? a.x : a.residual) + next * kP + k % kP;
        // the two halves of a 32-byte sector come by two copies: through L1, or each would fetch the sector (159 against 107 us)
        if (kP == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
      }
    }
    next += turn;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < kD; ++j) send(j);
  for (size_t g0 = (size_t)blockIdx.x * kThreads + threadIdx.x; g0 < groups; g0 += kD * turn) {
#pragma unroll
    for (int j = 0; j < kD; ++j) {
      const size_t g = g0 + j * turn;
      if (g >= groups) break;
      bool keep[kGroup];
      kept(g, a, keys, keep);
      asm volatile("cp.async.wait_group %0;" ::"n"(kD - 1) : "memory");
      uint4 xv[kP], rv[kP];
#pragma unroll
      for (int k = 0; k < kP; ++k) {
        xv[k] = ring[(j * kN * kP + k) * kThreads + threadIdx.x];
        if (kResidual) rv[k] = ring[(j * kN * kP + kP + k) * kThreads + threadIdx.x];
      }
      float f[kGroup], r[kGroup];
      unpack<T>(xv, f);
      if (kResidual) unpack<T>(rv, r);
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        f[i] = value(keep[i], f[i], a.scale);
        if (kResidual) f[i] = __fadd_rn(r[i], f[i]);
      }
      store(static_cast<T*>(a.y) + g * kGroup, f);
      send(j);
    }
  }
}

// Element by element: tensors that start anywhere, and (first > 0) the last, shorter group of the others.
template <typename T, bool kDeviceSeed>
__global__ void __launch_bounds__(kThreads) dropout_elements_kernel(const __grid_constant__ DropoutArgs a, size_t first) {
  pdl_prologue();
  Keys made;
  if (kDeviceSeed) make_keys(*a.seed_device, made);
  const Keys& keys = kDeviceSeed ? made : a.keys;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  for (size_t g = first + (size_t)blockIdx.x * kThreads + threadIdx.x; g < (a.n + kGroup - 1) / kGroup; g += (size_t)gridDim.x * kThreads) {
    bool keep[kGroup];
    kept(g, a, keys, keep);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      const size_t i = g * kGroup + j;
      if (i >= a.n) break;
      float v = value(keep[j], to_f(x[i]), a.scale);
      if (res) v = __fadd_rn(to_f(res[i]), v);
      from_f(static_cast<T*>(a.y)[i], v);
    }
  }
}

template <typename T, bool kDeviceSeed>
cudaError_t launch_dropout_t(const DropoutArgs& a, cudaStream_t stream) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const size_t cap = (size_t)sms * 16;      // a few rounds of what fits on the SMs at a time
  auto grid = [&](size_t groups) { const size_t b = (groups + kThreads - 1) / kThreads; return (unsigned)(b < cap ? b : cap); };
  const size_t all = (a.n + kGroup - 1) / kGroup, whole = al(a.x) && al(a.y) && al(a.residual) ? a.n / kGroup : 0;
  if (whole > 0) {
    const cudaError_t e = a.residual ? launch_after(dropout_kernel<T, true, kDeviceSeed>, grid(whole), kThreads, 0, stream, a)
                                     : launch_after(dropout_kernel<T, false, kDeviceSeed>, grid(whole), kThreads, 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  return whole < all ? launch_after(dropout_elements_kernel<T, kDeviceSeed>, grid(all - whole), kThreads, 0, stream, a, whole) : cudaSuccess;
}

}  // namespace
}  // namespace flame_b200

using namespace flame_b200;

extern "C" int flame_dropout(const void* x, const void* residual, void* y, size_t n, int dtype, double p, uint64_t seed,
                             const void* seed_device, uint64_t offset, void* stream) {
  const char* who = "flame_dropout";
  if (!(p >= 0.0 && p <= 1.0)) {
    set_last_error("flame_dropout: p must be in [0, 1]");
    return (int)cudaErrorInvalidValue;
  }
  if (dtype != FLAME_OFFLOAD_DTYPE_BF16 && dtype != FLAME_OFFLOAD_DTYPE_F32) {
    set_last_error("flame_dropout: dtype must be BF16 or F32");
    return (int)cudaErrorInvalidValue;
  }
  if (n == 0) return 0;
  auto al = [](const void* q, uintptr_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) == 0; };
  const uintptr_t size = dtype == FLAME_OFFLOAD_DTYPE_BF16 ? 2 : 4;
  if (!x || !y || !al(x, size) || !al(y, size) || !al(residual, size) || !al(seed_device, 8)) {
    set_last_error(!x || !y ? "flame_dropout: null tensor" : "flame_dropout: misaligned tensor");
    return (int)cudaErrorInvalidValue;
  }
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  const double t = nearbyint(p * 4294967296.0);   // 0 .. 2^32
  const uint64_t ti = (uint64_t)t;
  if (ti >> 32) {      // everything is dropped
    const size_t bytes = n * size;
    return cuda_result(who, residual ? cudaMemcpyAsync(y, residual, bytes, cudaMemcpyDeviceToDevice, (cudaStream_t)stream) : cudaMemsetAsync(y, 0, bytes, (cudaStream_t)stream));
  }
  DropoutArgs a;
  a.x = x; a.residual = residual; a.y = y; a.n = n;
  a.seed_device = static_cast<const uint64_t*>(seed_device);
  make_keys(seed, a.keys);
  a.o0 = (uint32_t)offset; a.o1 = (uint32_t)(offset >> 32);
  a.t_hi = (uint32_t)(ti >> 16); a.t_lo = (uint32_t)(ti & 0xFFFFu);
  a.scale = (float)(1.0 / (1.0 - p));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == FLAME_OFFLOAD_DTYPE_BF16) return cuda_result(who, seed_device ? launch_dropout_t<__nv_bfloat16, true>(a, s) : launch_dropout_t<__nv_bfloat16, false>(a, s));
  return cuda_result(who, seed_device ? launch_dropout_t<float, true>(a, s) : launch_dropout_t<float, false>(a, s));
}
