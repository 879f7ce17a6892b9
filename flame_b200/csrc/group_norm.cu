// Group norm with an activation on channels-last tensors, forward and backward, written for sm_100a.
//
//   x [B, L, C] BF16, G groups of C/G channels; per (sample, group) mean and variance over L x C/G elements;
//   h = (x - mean) * rstd * weight + bias, y = act(h), act = identity or silu(h) = h / (1 + exp(-h)).
//   backward: dh = dy * act'(h); db = sum dh, dw = sum dh * xhat over samples and positions;
//   s1 = sum of w*dh and s2 = sum of w*dh*xhat over the group; dx = rstd * (w*dh - (s1 + xhat*s2) / n).
//
// Two launches each way: the first reduces, the second applies.  A thread owns V neighbouring channels and walks down the
// positions of its chunk, so that a warp reads whole lines of the channels-last rows, and per-channel sums stay in registers.
// Sums are kept about a shift, the channel's first element in the sample: x - shift is of the size of the spread and not of the
// mean, so that sums of squares lose nothing when the mean is large against the spread.  A thread block turns its channel sums
// into (count, mean, sum of squares about the mean) of each group and writes those; the second launch joins the chunks' triples
// in a fixed order (T. Chan, G. Golub, R. LeVeque, 1983).  No atomics: the same inputs give the same bits.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "codec_kernels.cuh"
#include "common.h"
#include "fp8_device.cuh"

namespace flame_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct NormArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dy;       // backward
  const void* weight;            // NULL: 1
  const void* bias;              // NULL: 0
  __nv_bfloat16* y;              // forward: y, backward: dx
  uint8_t* codes;                // forward, may be NULL: FP8 codes of y, a scale for 128 elements of a row
  float* code_scales;
  float* stats;                  // [B, G, 2]: mean, rstd
  float* partial;                // forward: [B, parts, G, 3]; backward: [B, parts, G, 2]
  float* channel_partial;        // backward: [B, chunks, C, 2]
  void* dweight;                 // backward, may be NULL
  void* dbias;
  uint32_t B, C, G, cg;
  uint64_t L;
  uint32_t chunks;               // per sample
  uint64_t rows_per_chunk;
  uint32_t slabs;                // channel slabs of one thread block's width
  uint32_t slab_vecs;            // V-wide channel vectors in a slab
  float eps;
  int silu, params_f32;
};

__device__ __forceinline__ float param(const void* p, int f32, uint32_t c, float none) {
  if (!p) return none;
  return f32 ? static_cast<const float*>(p)[c] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
}
__device__ __forceinline__ float sigmoid(float h) { return __fdividef(1.0f, 1.0f + __expf(-h)); }

template <int V>
struct Vec { __nv_bfloat16 v[V]; };
template <>
struct alignas(16) Vec<8> { __nv_bfloat16 v[8]; };
template <>
struct alignas(4) Vec<2> { __nv_bfloat16 v[2]; };

template <int V>
__device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[V]) {
  const Vec<V> r = *reinterpret_cast<const Vec<V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = __bfloat162float(r.v[i]);
}
template <int V>
__device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[V]) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = __float2bfloat16_rn(f[i]);
  *reinterpret_cast<Vec<V>*>(p) = r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

// Where a thread works: which channel vector of the slab, which rows of the chunk.
template <int V>
struct Place {
  uint32_t b, chunk, slab, vec, lane_row, row_step, c0;
  uint64_t row0, row1;
  bool live;
  __device__ __forceinline__ explicit Place(const NormArgs& a) {
    chunk = blockIdx.x % a.chunks;
    const uint32_t rest = blockIdx.x / a.chunks;
    slab = rest % a.slabs;
    b = rest / a.slabs;
    const uint32_t nvec = a.C / V, first = slab * a.slab_vecs;
    const uint32_t here = nvec - first < a.slab_vecs ? nvec - first : a.slab_vecs;
    row_step = kThreads / here;
    vec = threadIdx.x % here;
    lane_row = threadIdx.x / here;
    live = lane_row < row_step;
    c0 = (first + vec) * V;
    row0 = (uint64_t)chunk * a.rows_per_chunk;
    row1 = row0 + a.rows_per_chunk < a.L ? row0 + a.rows_per_chunk : a.L;
  }
};

// Per-channel pairs of a thread block, added over its rows of threads in a fixed order: out[c] for the slab's channels.
template <int V>
__device__ __forceinline__ void join_rows(const Place<V>& p, const float (&s)[V], const float (&q)[V], float2* sh, uint32_t width) {
  // sh holds row_step x width pairs; width = channels of the slab
  if (p.live) {
#pragma unroll
    for (int i = 0; i < V; ++i) sh[p.lane_row * width + p.vec * V + i] = make_float2(s[i], q[i]);
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < width; c += kThreads) {
    float2 t = sh[c];
    for (uint32_t r = 1; r < p.row_step; ++r) {
      const float2 u = sh[r * width + c];
      t.x += u.x;
      t.y += u.y;
    }
    sh[c] = t;
  }
  __syncthreads();
}

template <int V>
__global__ void __launch_bounds__(kThreads) group_stats_kernel(const __grid_constant__ NormArgs a) {
  pdl_prologue();
  extern __shared__ float2 sh[];
  const Place<V> p(a);
  const __nv_bfloat16* xs = a.x + (size_t)p.b * a.L * a.C;
  float shift[V], s[V], q[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = q[i] = shift[i] = 0.0f;
  if (p.live) {
    load<V>(xs + p.c0, shift);
    for (uint64_t r = p.row0 + p.lane_row; r < p.row1; r += p.row_step) {
      float f[V];
      load<V>(xs + r * a.C + p.c0, f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = f[i] - shift[i];
        s[i] += d;
        q[i] = fmaf(d, d, q[i]);
      }
    }
  }
  const uint32_t slab_c0 = p.slab * a.slab_vecs * V;
  const uint32_t width = a.C - slab_c0 < a.slab_vecs * V ? a.C - slab_c0 : a.slab_vecs * V;
  join_rows<V>(p, s, q, sh, width);
  // a warp for each group: mean and sum of squares about it over the group's channels that lie in this slab
  const float n = (float)(p.row1 - p.row0);
  float* out = a.partial + ((size_t)(p.b * a.chunks + p.chunk) * a.slabs + p.slab) * a.G * 3;
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t g = threadIdx.x >> 5; g < a.G; g += kWarps) {
    const uint32_t lo = g * a.cg > slab_c0 ? g * a.cg : slab_c0;
    const uint32_t hi = (g + 1) * a.cg < slab_c0 + width ? (g + 1) * a.cg : slab_c0 + width;
    float count = 0.0f, mean = 0.0f, m2 = 0.0f;
    if (lo < hi && n > 0.0f) {
      float sum = 0.0f;
      for (uint32_t c = lo + lane; c < hi; c += 32) sum += __bfloat162float(xs[c]) + sh[c - slab_c0].x / n;
      mean = warp_sum(sum) / (float)(hi - lo);
      float acc = 0.0f;
      for (uint32_t c = lo + lane; c < hi; c += 32) {
        const float2 t = sh[c - slab_c0];
        const float off = __bfloat162float(xs[c]) + t.x / n - mean;
        acc += fmaxf(t.y - t.x * (t.x / n), 0.0f) + n * off * off;
      }
      m2 = warp_sum(acc);
      count = n * (float)(hi - lo);
    }
    if (lane == 0) { out[g * 3] = count; out[g * 3 + 1] = mean; out[g * 3 + 2] = m2; }
  }
}

// (mean, rstd) of every group of sample b, from the parts' triples: eight threads a group join every eighth part each, then
// their results, always in the same order.
__device__ __forceinline__ void chan(float& n, float& mean, float& m2, float n2, float mean2, float m22) {
  const float t = n + n2;
  if (n2 <= 0.0f) return;
  if (n <= 0.0f) { n = n2; mean = mean2; m2 = m22; return; }
  const float d = mean2 - mean, f = n2 / t;
  mean = fmaf(d, f, mean);
  m2 += m22 + d * d * n * f;
  n = t;
}
__device__ __forceinline__ void finish_stats(const NormArgs& a, uint32_t b, float2* stats) {
  const uint32_t parts = a.chunks * a.slabs;
  for (uint32_t g0 = 0; g0 < a.G; g0 += kThreads / 8) {
    const uint32_t g = g0 + threadIdx.x / 8, k = threadIdx.x % 8;
    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    if (g < a.G) {
      const float* in = a.partial + ((size_t)b * parts * a.G + g) * 3;
      for (uint32_t i = k; i < parts; i += 8) {
        const float* t = in + (size_t)i * a.G * 3;
        chan(n, mean, m2, t[0], t[1], t[2]);
      }
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
      const float n2 = __shfl_xor_sync(0xFFFFFFFFu, n, d), e2 = __shfl_xor_sync(0xFFFFFFFFu, mean, d), v2 = __shfl_xor_sync(0xFFFFFFFFu, m2, d);
      if (k & d) { float na = n2, ma = e2, va = v2; chan(na, ma, va, n, mean, m2); n = na; mean = ma; m2 = va; }
      else chan(n, mean, m2, n2, e2, v2);
    }
    if (g < a.G && k == 0) stats[g] = make_float2(mean, rsqrtf(m2 / n + a.eps));
  }
  __syncthreads();
}

// Codes of V = 8 channels a thread, 16 threads hold a block of 128 channels of a row (C a multiple of 128).
__device__ __forceinline__ uint2 encode_row_block(const float (&y)[8], float& scale) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));   // a NaN is ignored
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
  scale = fp8_scale_of(amax);
  return fp8_encode8(y, scale, fp8_factor_of(scale));
}

template <int V, bool kCodes>
__global__ void __launch_bounds__(kThreads) group_apply_kernel(const __grid_constant__ NormArgs a) {
  pdl_prologue();
  extern __shared__ float2 sh[];
  const Place<V> p(a);
  finish_stats(a, p.b, sh);
  if (p.chunk == 0 && p.slab == 0)
    for (uint32_t g = threadIdx.x; g < a.G; g += kThreads) {
      a.stats[((size_t)p.b * a.G + g) * 2] = sh[g].x;
      a.stats[((size_t)p.b * a.G + g) * 2 + 1] = sh[g].y;
    }
  float mean[V], scale[V], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t c = p.c0 + i;
    mean[i] = scale[i] = bias[i] = 0.0f;
    if (p.live) {
      const float2 t = sh[c / a.cg];
      mean[i] = t.x;
      scale[i] = t.y * param(a.weight, a.params_f32, c, 1.0f);
      bias[i] = param(a.bias, a.params_f32, c, 0.0f);
    }
  }
  const size_t base = (size_t)p.b * a.L * a.C;
  // with codes, 16 neighbouring lanes share a row: C / 8 is a multiple of 16 and so is the slab's width, so they are all live or none is
  for (uint64_t r0 = p.row0; r0 < p.row1; r0 += p.row_step) {
    const uint64_t r = r0 + p.lane_row;
    const bool in = p.live && r < p.row1;
    if (!kCodes && !in) continue;
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = 0.0f;
    const size_t at = base + r * a.C + p.c0;
    if (in) load<V>(a.x + at, f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float h = fmaf(f[i] - mean[i], scale[i], bias[i]);
      f[i] = a.silu ? h * sigmoid(h) : h;
    }
    if (in) store<V>(a.y + at, f);
    if constexpr (kCodes) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __bfloat162float(__float2bfloat16_rn(f[i]));   // the codes are those of the BF16 output
      float s;
      const uint2 c = encode_row_block(f, s);
      if (in) {
        *reinterpret_cast<uint2*>(a.codes + at) = c;
        if ((p.vec & 15) == 0) a.code_scales[at / 128] = s;
      }
    }
  }
}

// dh = dy * act'(h) of V channels
template <int V>
__device__ __forceinline__ void grad_h(const float (&x)[V], const float (&dy)[V], const float (&mean)[V], const float (&rstd)[V],
                                       const float (&w)[V], const float (&bias)[V], int silu, float (&xhat)[V], float (&dh)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    xhat[i] = (x[i] - mean[i]) * rstd[i];
    dh[i] = dy[i];
    if (silu) {
      const float h = fmaf(xhat[i], w[i], bias[i]), g = sigmoid(h);
      dh[i] *= g * fmaf(h, 1.0f - g, 1.0f);
    }
  }
}

template <int V>
__device__ __forceinline__ void channel_params(const NormArgs& a, const Place<V>& p, float (&mean)[V], float (&rstd)[V], float (&w)[V], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mean[i] = rstd[i] = w[i] = bias[i] = 0.0f;
    if (p.live) {
      const uint32_t c = p.c0 + i;
      const float* t = a.stats + ((size_t)p.b * a.G + c / a.cg) * 2;
      mean[i] = t[0];
      rstd[i] = t[1];
      w[i] = param(a.weight, a.params_f32, c, 1.0f);
      bias[i] = param(a.bias, a.params_f32, c, 0.0f);
    }
  }
}

template <int V>
__global__ void __launch_bounds__(kThreads) group_grad_sums_kernel(const __grid_constant__ NormArgs a) {
  pdl_prologue();
  extern __shared__ float2 sh[];
  const Place<V> p(a);
  float mean[V], rstd[V], w[V], bias[V], s[V], q[V];
  channel_params<V>(a, p, mean, rstd, w, bias);
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = q[i] = 0.0f;
  const size_t base = (size_t)p.b * a.L * a.C;
  if (p.live) {
    for (uint64_t r = p.row0 + p.lane_row; r < p.row1; r += p.row_step) {
      float x[V], dy[V], xhat[V], dh[V];
      load<V>(a.x + base + r * a.C + p.c0, x);
      load<V>(a.dy + base + r * a.C + p.c0, dy);
      grad_h<V>(x, dy, mean, rstd, w, bias, a.silu, xhat, dh);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] += dh[i];
        q[i] = fmaf(dh[i], xhat[i], q[i]);
      }
    }
  }
  const uint32_t slab_c0 = p.slab * a.slab_vecs * V;
  const uint32_t width = a.C - slab_c0 < a.slab_vecs * V ? a.C - slab_c0 : a.slab_vecs * V;
  join_rows<V>(p, s, q, sh, width);
  float2* cp = reinterpret_cast<float2*>(a.channel_partial) + (size_t)(p.b * a.chunks + p.chunk) * a.C + slab_c0;
  for (uint32_t c = threadIdx.x; c < width; c += kThreads) cp[c] = sh[c];
  float* out = a.partial + ((size_t)(p.b * a.chunks + p.chunk) * a.slabs + p.slab) * a.G * 2;
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t g = threadIdx.x >> 5; g < a.G; g += kWarps) {
    const uint32_t lo = g * a.cg > slab_c0 ? g * a.cg : slab_c0;
    const uint32_t hi = (g + 1) * a.cg < slab_c0 + width ? (g + 1) * a.cg : slab_c0 + width;
    float s1 = 0.0f, s2 = 0.0f;
    for (uint32_t c = lo + lane; c < hi; c += 32) {
      const float wc = param(a.weight, a.params_f32, c, 1.0f);
      s1 = fmaf(wc, sh[c - slab_c0].x, s1);
      s2 = fmaf(wc, sh[c - slab_c0].y, s2);
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (lane == 0) { out[g * 2] = s1; out[g * 2 + 1] = s2; }
  }
}

// The first blocks apply; the blocks behind them add the channel sums up to dweight and dbias.
template <int V>
__global__ void __launch_bounds__(kThreads) group_grad_apply_kernel(const __grid_constant__ NormArgs a, uint32_t apply_blocks) {
  pdl_prologue();
  extern __shared__ float2 sh[];
  if (blockIdx.x >= apply_blocks) {
    // a warp's 32 lanes take 32 neighbouring channels, the eight warps every eighth part
    __shared__ float2 part[kWarps][32];
    const uint32_t lane = threadIdx.x & 31, wp = threadIdx.x >> 5, c = (blockIdx.x - apply_blocks) * 32 + lane;
    const float2* cp = reinterpret_cast<const float2*>(a.channel_partial);
    const uint32_t parts = a.B * a.chunks;
    float2 t = make_float2(0.0f, 0.0f);
    if (c < a.C)
      for (uint32_t i = wp; i < parts; i += kWarps) {
        const float2 u = cp[(size_t)i * a.C + c];
        t.x += u.x;
        t.y += u.y;
      }
    part[wp][lane] = t;
    __syncthreads();
    if (wp == 0 && c < a.C) {
      for (int k = 1; k < kWarps; ++k) { t.x += part[k][lane].x; t.y += part[k][lane].y; }
      if (a.params_f32) {
        if (a.dbias) static_cast<float*>(a.dbias)[c] = t.x;
        if (a.dweight) static_cast<float*>(a.dweight)[c] = t.y;
      } else {
        if (a.dbias) static_cast<__nv_bfloat16*>(a.dbias)[c] = __float2bfloat16_rn(t.x);
        if (a.dweight) static_cast<__nv_bfloat16*>(a.dweight)[c] = __float2bfloat16_rn(t.y);
      }
    }
    return;
  }
  const Place<V> p(a);
  {
    const uint32_t parts = a.chunks * a.slabs;
    const float inv_n = 1.0f / ((float)a.L * (float)a.cg);
    for (uint32_t g0 = 0; g0 < a.G; g0 += kThreads / 8) {
      const uint32_t g = g0 + threadIdx.x / 8, k = threadIdx.x % 8;
      float s1 = 0.0f, s2 = 0.0f;
      if (g < a.G) {
        const float* in = a.partial + ((size_t)p.b * parts * a.G + g) * 2;
        for (uint32_t i = k; i < parts; i += 8) {
          s1 += in[(size_t)i * a.G * 2];
          s2 += in[(size_t)i * a.G * 2 + 1];
        }
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) {
        s1 += __shfl_xor_sync(0xFFFFFFFFu, s1, d);
        s2 += __shfl_xor_sync(0xFFFFFFFFu, s2, d);
      }
      if (g < a.G && k == 0) sh[g] = make_float2(s1 * inv_n, s2 * inv_n);
    }
    __syncthreads();
  }
  float mean[V], rstd[V], w[V], bias[V], m1[V], m2[V];
  channel_params<V>(a, p, mean, rstd, w, bias);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 t = p.live ? sh[(p.c0 + i) / a.cg] : make_float2(0.0f, 0.0f);
    m1[i] = t.x;
    m2[i] = t.y;
  }
  const size_t base = (size_t)p.b * a.L * a.C;
  if (!p.live) return;
  for (uint64_t r = p.row0 + p.lane_row; r < p.row1; r += p.row_step) {
    float x[V], dy[V], xhat[V], dh[V];
    const size_t at = base + r * a.C + p.c0;
    load<V>(a.x + at, x);
    load<V>(a.dy + at, dy);
    grad_h<V>(x, dy, mean, rstd, w, bias, a.silu, xhat, dh);
#pragma unroll
    for (int i = 0; i < V; ++i) dh[i] = rstd[i] * (fmaf(w[i], dh[i], -m1[i]) - xhat[i] * m2[i]);
    store<V>(a.y + at, dh);
  }
}

int sm_count_here() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// How a call is cut: the width of a thread's channel vector, slabs of channels, chunks of positions.
struct Plan {
  int V;
  uint32_t slab_vecs, slabs, chunks;
  uint64_t rows_per_chunk;
};
Plan plan(uint32_t B, uint64_t L, uint32_t C, bool aligned16, bool aligned4, int sms) {
  Plan p;
  p.V = (C % 8 == 0 && aligned16) ? 8 : (C % 2 == 0 && aligned4) ? 2 : 1;
  const uint32_t nvec = C / p.V;
  p.slabs = (nvec + kThreads - 1) / kThreads;
  // with slabs, a width that is a multiple of 16 vectors: a block of 128 channels lies in one slab
  p.slab_vecs = p.slabs == 1 ? nvec : kThreads;
  // about four thread blocks on each SM, and at least 16 rows of threads' worth of work in a chunk
  const uint64_t want = ((uint64_t)sms * 4 + (uint64_t)B * p.slabs - 1) / ((uint64_t)B * p.slabs);
  const uint32_t row_step = kThreads / p.slab_vecs;
  uint64_t most = (L + (uint64_t)row_step * 4 - 1) / ((uint64_t)row_step * 4);
  if (most < 1) most = 1;
  uint64_t chunks = want < most ? want : most;
  if (chunks < 1) chunks = 1;
  if (chunks > 1024) chunks = 1024;
  p.rows_per_chunk = (L + chunks - 1) / chunks;
  if (p.rows_per_chunk < 1) p.rows_per_chunk = 1;
  p.chunks = (uint32_t)((L + p.rows_per_chunk - 1) / p.rows_per_chunk);
  if (p.chunks < 1) p.chunks = 1;
  return p;
}
size_t partial_floats(const Plan& p, uint32_t B, uint32_t C, uint32_t G, bool backward) {
  const size_t groups = (size_t)B * p.chunks * p.slabs * G * (backward ? 2 : 3);
  return ((groups + 3) / 4 * 4) + (backward ? (size_t)B * p.chunks * C * 2 : 0);
}
bool al(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check(const char* who, uint64_t B, uint64_t L, uint64_t C, uint64_t G, int activation, int param_dtype) {
  const char* what = nullptr;
  if (G == 0 || C == 0 || C % G != 0) what = "the channels must be a positive multiple of the groups";
  else if (C > 65536) what = "at most 65536 channels";
  else if (G > 4096) what = "at most 4096 groups";
  else if (B > 65535 || L > 0x7FFFFFFFull) what = "at most 65535 samples of at most 2^31 - 1 positions";
  else if (activation != FLAME_ACTIVATION_NONE && activation != FLAME_ACTIVATION_SILU) what = "unknown activation";
  else if (param_dtype != FLAME_OFFLOAD_DTYPE_BF16 && param_dtype != FLAME_OFFLOAD_DTYPE_F32) what = "weight and bias must be BF16 or F32";
  if (!what) return 0;
  set_last_error(std::string(who) + ": " + what);
  return (int)cudaErrorInvalidValue;
}
int refuse(const char* who, const char* what) {
  set_last_error(std::string(who) + ": " + what);
  return (int)cudaErrorInvalidValue;
}

template <typename F>
cudaError_t by_width(int V, F&& f) {
  if (V == 8) return f(std::integral_constant<int, 8>());
  if (V == 2) return f(std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 1>());
}

}  // namespace
}  // namespace flame_b200

using namespace flame_b200;

extern "C" {

size_t flame_group_norm_workspace_bytes(size_t B, size_t L, size_t C, size_t G, int backward) {
  if (check("flame_group_norm_workspace_bytes", B, L, C, G, 0, 0) != 0 || B == 0 || L == 0) return 0;
  size_t most = 0;   // whatever the alignment of the tensors turns out to be
  for (int k = 0; k < 3; ++k) {
    const size_t f = partial_floats(plan((uint32_t)B, L, (uint32_t)C, k == 0, k <= 1, sm_count_here()), (uint32_t)B, (uint32_t)C, (uint32_t)G, backward != 0);
    most = f > most ? f : most;
  }
  return most * sizeof(float);
}

int flame_group_norm(const void* x, const void* weight, const void* bias, void* y, void* codes, void* code_scales, void* stats,
                     size_t B, size_t L, size_t C, size_t G, float eps, int activation, int param_dtype, void* workspace,
                     size_t workspace_bytes, void* stream) {
  const char* who = "flame_group_norm";
  if (const int e = check(who, B, L, C, G, activation, param_dtype)) return e;
  if (B == 0 || L == 0) return 0;
  if (!x || !y || !stats || !workspace) return refuse(who, "null tensor");
  if (workspace_bytes < flame_group_norm_workspace_bytes(B, L, C, G, 0)) return refuse(who, "workspace too small");
  if (!al(x, 2) || !al(y, 2) || !al(stats, 4) || !al(workspace, 16)) return refuse(who, "misaligned tensor");
  const bool al16 = al(x, 16) && al(y, 16);
  if (codes && (C % 128 != 0 || !al16 || !al(codes, 8) || !code_scales)) return refuse(who, "codes need channels % 128 == 0, 16-byte aligned tensors and a place for the scales");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return (int)cudaErrorLaunchFailure;
  const Plan p = plan((uint32_t)B, L, (uint32_t)C, al16, al(x, 4) && al(y, 4), sm_count_here());
  NormArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.weight = weight; a.bias = bias; a.y = static_cast<__nv_bfloat16*>(y);
  a.codes = static_cast<uint8_t*>(codes); a.code_scales = static_cast<float*>(code_scales); a.stats = static_cast<float*>(stats);
  a.partial = static_cast<float*>(workspace);
  a.B = (uint32_t)B; a.C = (uint32_t)C; a.G = (uint32_t)G; a.cg = (uint32_t)(C / G); a.L = L;
  a.chunks = p.chunks; a.rows_per_chunk = p.rows_per_chunk; a.slabs = p.slabs; a.slab_vecs = p.slab_vecs;
  a.eps = eps; a.silu = activation == FLAME_ACTIVATION_SILU; a.params_f32 = param_dtype == FLAME_OFFLOAD_DTYPE_F32;
  const unsigned grid = (unsigned)(B * p.slabs * p.chunks);
  const size_t sums = (size_t)kThreads * p.V * sizeof(float2), groups = G * sizeof(float2);
  cudaStream_t s = (cudaStream_t)stream;
  return (int)by_width(p.V, [&](auto v) {
    constexpr int V = decltype(v)::value;
    cudaError_t e = launch_after(group_stats_kernel<V>, grid, kThreads, sums, s, a);
    if (e != cudaSuccess) return e;
    if constexpr (V == 8) {
      if (a.codes) return launch_after(group_apply_kernel<8, true>, grid, kThreads, groups, s, a);
    }
    return launch_after(group_apply_kernel<V, false>, grid, kThreads, groups, s, a);
  });
}

int flame_group_norm_backward(const void* x, const void* dy, const void* weight, const void* bias, const void* stats, void* dx,
                              void* dweight, void* dbias, size_t B, size_t L, size_t C, size_t G, int activation, int param_dtype,
                              void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "flame_group_norm_backward";
  if (const int e = check(who, B, L, C, G, activation, param_dtype)) return e;
  cudaStream_t s = (cudaStream_t)stream;
  const size_t psize = param_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2;
  if (B == 0 || L == 0) {   // sums over nothing
    if (dweight) if (const cudaError_t e = cudaMemsetAsync(dweight, 0, C * psize, s)) return (int)e;
    if (dbias) if (const cudaError_t e = cudaMemsetAsync(dbias, 0, C * psize, s)) return (int)e;
    return 0;
  }
  if (!x || !dy || !dx || !stats || !workspace) return refuse(who, "null tensor");
  if (workspace_bytes < flame_group_norm_workspace_bytes(B, L, C, G, 1)) return refuse(who, "workspace too small");
  if (!al(x, 2) || !al(dy, 2) || !al(dx, 2) || !al(stats, 4) || !al(workspace, 16)) return refuse(who, "misaligned tensor");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return (int)cudaErrorLaunchFailure;
  const Plan p = plan((uint32_t)B, L, (uint32_t)C, al(x, 16) && al(dy, 16) && al(dx, 16), al(x, 4) && al(dy, 4) && al(dx, 4), sm_count_here());
  NormArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.dy = static_cast<const __nv_bfloat16*>(dy); a.weight = weight; a.bias = bias;
  a.y = static_cast<__nv_bfloat16*>(dx); a.stats = const_cast<float*>(static_cast<const float*>(stats));
  a.partial = static_cast<float*>(workspace);
  a.channel_partial = a.partial + ((size_t)B * p.chunks * p.slabs * G * 2 + 3) / 4 * 4;
  a.dweight = dweight; a.dbias = dbias;
  a.B = (uint32_t)B; a.C = (uint32_t)C; a.G = (uint32_t)G; a.cg = (uint32_t)(C / G); a.L = L;
  a.chunks = p.chunks; a.rows_per_chunk = p.rows_per_chunk; a.slabs = p.slabs; a.slab_vecs = p.slab_vecs;
  a.silu = activation == FLAME_ACTIVATION_SILU; a.params_f32 = param_dtype == FLAME_OFFLOAD_DTYPE_F32;
  const unsigned grid = (unsigned)(B * p.slabs * p.chunks);
  const unsigned more = (dweight || dbias) ? (unsigned)((C + 31) / 32) : 0;
  const size_t sums = (size_t)kThreads * p.V * sizeof(float2), groups = G * sizeof(float2);
  return (int)by_width(p.V, [&](auto v) {
    constexpr int V = decltype(v)::value;
    const cudaError_t e = launch_after(group_grad_sums_kernel<V>, grid, kThreads, sums, s, a);
    if (e != cudaSuccess) return e;
    return launch_after(group_grad_apply_kernel<V>, grid + more, kThreads, groups, s, a, (uint32_t)grid);
  });
}

}  // extern "C"
