// Group norm with an activation on channels-last tensors, forward and backward, written for sm_100a.
//
//   x [B, L, C] BF16, G groups of C/G channels; per (sample, group) mean and variance over L x C/G elements;
//   h = (x - mean) * rstd * weight + bias, y = act(h), act = identity or silu(h) = h / (1 + exp(-h)).
//   backward: dh = dy * act'(h); db = sum dh, dw = sum dh * xhat over samples and positions;
//   s1 = sum of w*dh and s2 = sum of w*dh*xhat over the group; dx = rstd * (w*dh - (s1 + xhat*s2) / n).
//
// Two launches each way: the first reduces, the second applies.  A thread owns V neighbouring channels and walks down the
// positions of its chunk, so that a warp reads whole lines of the channels-last rows, and per-channel sums stay in registers.
// A block's forward sums are kept about a shift, the median of the group's first elements in the first, middle and last row of its chunk:
// x - shift is of the size of the spread and not of the mean, so that sums of squares lose nothing when the mean is large against the
// spread.  (The first element alone may be an outlier, at a distance D from the others: the chunk's n elements, some thousands, then
// sum to n D^2 and err by n 2^-24 D^2, where the outlier's own share of the variance is D^2.)  Blocks are then joined by their mean and sum of
// squares about it (T. Chan, G. Golub, R. LeVeque, 1983): a cluster's through distributed shared memory, which leaves the second
// launch a quarter of them to read; where there are many, a launch of a block for each group joins them in between.  Everything is
// added in a fixed order, without atomics: the same inputs give the same bits.
//
// What bounds it, measured on one B200 (calls recorded in a CUDA graph and replayed back to back): memory where x is larger than the L2
// cache, which the second launch then reads again (1024 x 1024 x 128 with silu: forward 139 us for 537 MB in and out and 268 read twice,
// 5.8 TB/s; with codes 191 us; 1 x 524288 x 128 forward and backward 203 us); the way through two dependent launches and their joins where it is
// small (1 x 64 x 1280 forward 9.1 us, and backward 20.1; 4 x 4096 x 320 15.2 and 34.5; of those 8 us a launch some 3 are the rows, 2 the
// cluster's join, 2 the joining of the parts).
//
// Squares are binary32 numbers: a group with values further than 1e19 from the others has NaN.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "codec_kernels.cuh"
#include "common.h"
#include "fp8_device.cuh"

namespace flame_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kCluster = 4;
// Over 64 parts the blocks of the second launch would spend longer on joining them than a launch between the two takes.
constexpr uint32_t kMostParts = 64;

struct NormArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dy;       // backward
  const void* weight;            // NULL: 1
  const void* bias;              // NULL: 0
  __nv_bfloat16* y;              // forward: y, backward: dx
  uint8_t* codes;                // forward, may be NULL: FP8 codes of y, a scale for 128 elements of a row
  float* code_scales;
  float* stats;                  // [B, G, 2]: mean, rstd
  float2* partial;               // [B, parts, G]: forward mean and sum of squares about it, backward s1 and s2
  float2* channel_partial;       // backward: [B, parts, C]: sums for dbias and dweight
  float2* finished;              // NULL, or [B, G]: what the launch between the two made of the parts
  void* dweight;                 // backward, may be NULL
  void* dbias;
  uint32_t B, C, G, cg, by_cg;
  uint64_t L;
  uint32_t chunks;               // per sample and slab, a multiple of the cluster's blocks (the last ones may be empty)
  uint32_t parts;                // clusters per sample: chunks / kCluster * slabs
  uint32_t rows_per_chunk;
  uint32_t slabs;                // channel slabs of one thread block's width
  uint32_t slab_vecs, V;         // V-wide channel vectors in a slab
  float eps;
  int silu, params_f32;
  int stream;                    // x and y together are larger than the L2 cache
};

__device__ __forceinline__ float param(const void* p, int f32, uint32_t c, float none) {
  if (!p) return none;
  return f32 ? static_cast<const float*>(p)[c] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
}
// Two binary32 numbers in one register pair: additions and multiply-adds take one instruction for both.
struct F2 {
  uint64_t v;
  F2() = default;
  __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ float2 get() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ F2 add(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 mul(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }

// 1 / (1 + exp(-h)) of two numbers on the special-function unit, which is what bounds the kernels next to memory (16 results a cycle
// and SM): two exponentials and one reciprocal, of the product, from which each takes its own.  The exponentials end at 2^60, so
// that the product stays finite, and a little more than 2^-60 is taken off every result, which saturates: under h = -60 ln 2 = -41.6 it is
// 0, so that h times it vanishes however far below zero h is (a channel that its bias masks), with an error of 42 * 2^-60 at most.  (A
// comparison and a selection for each result took 2 % longer at 4 x 4096 x 320.)  A NaN counts as 60 too: it would make its neighbour NaN,
// which may belong to another group, and comes back by the factor h that every use has, as does the NaN of -infinity times 0.  Above
// -41.6 the rounding of t decides, |t| 2^-24 of the result, 2^-18 at most: below the 2^-8 of the rounding to BF16.
__device__ __forceinline__ F2 sigmoid(F2 h) {
  const float2 t = mul(h, F2(-1.442695041f, -1.442695041f)).get();
  float e0, e1, r, g0, g1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(fminf(t.x, 60.0f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(fminf(t.y, 60.0f)));
  const float2 a = add(F2(e0, e1), F2(1.0f, 1.0f)).get();
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a.x * a.y));
  constexpr float kOff = -(1.0f + 0x1p-16f) * 0x1p-60f;      // the results err by 2^-22 of themselves
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(g0) : "f"(r), "f"(a.y), "f"(kOff));
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(g1) : "f"(r), "f"(a.x), "f"(kOff));
  return F2(g0, g1);
}
// The group of channel c: c / cg by a multiplication, exact for c and cg up to 65,536 (by_cg = ceil(2^32 / cg), 0 for cg = 1).
// Eight divisions a thread took longer than the sums themselves at 64 x 64 positions.
__device__ __forceinline__ uint32_t group_of(uint32_t c, uint32_t by_cg) { return by_cg ? __umulhi(c, by_cg) : c; }

template <int V>
struct Vec { __nv_bfloat16 v[V]; };
template <>
struct alignas(16) Vec<8> { __nv_bfloat16 v[8]; };
template <>
struct alignas(4) Vec<2> { __nv_bfloat16 v[2]; };

// Pairs of neighbouring channels; with one channel the pair's other half is 0.
template <int V>
constexpr int kPairs = (V + 1) / 2;
template <int V>
__device__ __forceinline__ void unpack(const Vec<V>& r, F2 (&f)[kPairs<V>]) {
  if constexpr (V == 1) {
    f[0] = F2(__bfloat162float(r.v[0]), 0.0f);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(&r)[i];
      f[i] = F2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
  }
}
__device__ __forceinline__ uint32_t to_bf16x2(F2 f) {
  const float2 u = f.get();
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(u.y), "f"(u.x));
  return w;
}
template <int V>
__device__ __forceinline__ void store(__nv_bfloat16* p, const F2 (&f)[kPairs<V>], int stream) {
  if constexpr (V == 8) {
    const uint4 w = make_uint4(to_bf16x2(f[0]), to_bf16x2(f[1]), to_bf16x2(f[2]), to_bf16x2(f[3]));
    if (stream) __stcs(reinterpret_cast<uint4*>(p), w);
    else *reinterpret_cast<uint4*>(p) = w;
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint32_t*>(p) = to_bf16x2(f[0]);
  } else {
    *p = __float2bfloat16_rn(f[0].get().x);
  }
}

// A thread's way down its rows, kN tensors at a time; kBack: from the last row to the first.  The constructor sends the first rows on
// their way, run(f) calls f(offset, vectors) for each row, offset in elements from the thread's first row.
//
// The rows ahead are on their way to shared memory as asynchronous copies, each thread's own in places of its own, so nothing waits
// for another thread and nothing is held in registers: with one row in flight in registers the two passes over 1024 x 1024 x 128
// took 72 and 174 us, with four, which left two blocks on an SM, 76 and 152, this way 57 and 95 (before what came later).
constexpr int kDepth = 8;
constexpr size_t kRingBytes = (size_t)kDepth * kThreads * 16;
constexpr uint32_t kMostGroups = 4096;
constexpr int kMostShared = (int)(kRingBytes + (kThreads * 8 + kMostGroups) * sizeof(float2) + kMostGroups * sizeof(float));
template <int kN, int V, bool kBack>
struct Walk {
  [[maybe_unused]] static constexpr int kD = V == 8 ? kDepth / kN : 1;      // rows on their way
  const __nv_bfloat16* const (&src)[kN];
  uint4* ring;
  uint32_t mine, at_shared;
  ptrdiff_t step, first, next;

  // the row of round n, into place j of the ring
  __device__ __forceinline__ void send(uint32_t n, int j) {
    if (n < mine) {
#pragma unroll
      for (int k = 0; k < kN; ++k)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at_shared + (j * kN + k) * kThreads * 16), "l"(src[k] + next) : "memory");
    }
    next += step;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ Walk(const __nv_bfloat16* const (&s)[kN], uint32_t rows, uint32_t lane_row, uint32_t row_step, uint32_t C, uint4* r) : src(s), ring(r) {
    mine = rows > lane_row ? (rows - lane_row + row_step - 1) / row_step : 0;
    step = (kBack ? -1 : 1) * (ptrdiff_t)((size_t)row_step * C);
    first = next = kBack ? -step * ((ptrdiff_t)mine - 1) : 0;
    at_shared = (uint32_t)__cvta_generic_to_shared(ring + threadIdx.x);
    if constexpr (V == 8) {
#pragma unroll
      for (int j = 0; j < kD; ++j) send(j, j);
    }
  }
  template <typename F>
  __device__ __forceinline__ void run(F&& f) {
    ptrdiff_t at = first;
    if constexpr (V == 8) {
      for (uint32_t n0 = 0; n0 < mine; n0 += kD) {
#pragma unroll
        for (int j = 0; j < kD; ++j) {      // a turn of the ring
          if (n0 + j >= mine) break;
          asm volatile("cp.async.wait_group %0;" ::"n"(kD - 1) : "memory");
          Vec<V> v[kN];
#pragma unroll
          for (int k = 0; k < kN; ++k) { const uint4 w = ring[(j * kN + k) * kThreads + threadIdx.x]; v[k] = *reinterpret_cast<const Vec<V>*>(&w); }
          f(at, v);
          at += step;
          send(n0 + j + kD, j);
        }
      }
    } else {
      for (uint32_t n = 0; n < mine; ++n, at += step) {
        Vec<V> v[kN];
#pragma unroll
        for (int k = 0; k < kN; ++k) v[k] = *reinterpret_cast<const Vec<V>*>(src[k] + at);
        f(at, v);
      }
    }
  }
};

// V neighbouring channels of weight or bias
template <int V>
__device__ __forceinline__ void params(const void* p, int f32, uint32_t c, float none, float (&out)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = none;
  if (V == 8 && p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {      // c is a multiple of 8
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + c);
    float4 lo, hi;
    if (f32) {
      lo = f[0];
      hi = f[1];
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + c);
      lo = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
      hi = make_float4(__uint_as_float(w.z << 16), __uint_as_float(w.z & 0xFFFF0000u), __uint_as_float(w.w << 16), __uint_as_float(w.w & 0xFFFF0000u));
    }
    const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = v[i];
  } else if (p && f32) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = static_cast<const float*>(p)[c + i];
  } else if (p) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c + i]);
  }
}

// Shared memory: the ring (vectors of eight channels only), then pairs of sums.
template <int V>
__device__ __forceinline__ float2* sums_of(uint4* ring) { return reinterpret_cast<float2*>(ring + (V == 8 ? kRingBytes / 16 : 0)); }

// Where a thread works: which channel vector of the slab, which rows of the chunk.
template <int V>
struct Place {
  uint32_t b, chunk, slab, vec, lane_row, row_step, c0;
  uint64_t row0;
  uint32_t rows;
  bool live;
  // back: the last chunk first, which the launch before has read last
  __device__ __forceinline__ explicit Place(const NormArgs& a, bool back = false) {
    chunk = back ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    slab = blockIdx.y;
    b = blockIdx.z;
    const uint32_t nvec = a.C / V, first = slab * a.slab_vecs;
    const uint32_t here = nvec - first < a.slab_vecs ? nvec - first : a.slab_vecs;
    row_step = kThreads / here;
    lane_row = threadIdx.x / here;
    vec = threadIdx.x - lane_row * here;
    live = lane_row < row_step;
    c0 = (first + vec) * V;
    row0 = (uint64_t)chunk * a.rows_per_chunk;
    if (row0 > a.L) row0 = a.L;
    rows = a.L - row0 < a.rows_per_chunk ? (uint32_t)(a.L - row0) : a.rows_per_chunk;
  }
};

// Per-channel pairs of a thread block, added over its rows of threads in a fixed order.  Channel c of the slab lies at
// place_of(c): first every vector's first channel, then every second one, so that neighbouring lanes write neighbouring words.
template <int V>
__device__ __forceinline__ uint32_t place_of(uint32_t c, uint32_t width) { return c % V * (width / V) + c / V; }
template <int V>
__device__ __forceinline__ void join_rows(const Place<V>& p, const F2 (&s)[kPairs<V>], const F2 (&q)[kPairs<V>], float2* sh, uint32_t width) {
  // sh holds row_step x width pairs; width = channels of the slab
  if (p.live) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 si = s[i / 2].get(), qi = q[i / 2].get();
      sh[p.lane_row * width + i * (width / V) + p.vec] = i % 2 ? make_float2(si.y, qi.y) : make_float2(si.x, qi.x);
    }
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

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// `count` pairs of every block's `sh`, pair i at place(i), joined over the cluster's blocks in the order of their ranks; each block
// joins and writes its share.  Between two cluster_sync_all(): the pairs are there, and nobody leaves or writes them while they are read.
template <typename F, typename J>
__device__ __forceinline__ void join_cluster(const float2* sh, uint32_t count, float2* out, F&& place, J&& join) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(sh));
  for (uint32_t i = cluster_rank() + kCluster * threadIdx.x; i < count; i += kCluster * kThreads) {
    float2 v[kCluster];
#pragma unroll
    for (uint32_t k = 0; k < kCluster; ++k) {
      uint32_t peer;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at + place(i) * 8), "r"(k));
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[k].x), "=f"(v[k].y) : "r"(peer) : "memory");
    }
    out[i] = join(i, v);
  }
}
__device__ __forceinline__ float2 add_up(const float2 (&v)[kCluster]) {
  float2 t = v[0];
#pragma unroll
  for (uint32_t k = 1; k < kCluster; ++k) { t.x += v[k].x; t.y += v[k].y; }
  return t;
}
// The slab's channel sums, weighted, added up to the groups that the slab touches: one, eight or 32 lanes a group.  (20 channels took
// one thread 1.2 us, 30 cycles for each word from shared memory.)
template <typename F, typename D>
__device__ __forceinline__ void join_channels(const NormArgs& a, uint32_t slab_c0, uint32_t width, float2* groups, F&& pair, D&& done) {
  const uint32_t lanes = a.cg > 32 ? 32 : a.cg > 8 ? 8 : 1, lane = threadIdx.x & (lanes - 1);
  for (uint32_t g0 = 0; g0 < a.G; g0 += kThreads / lanes) {
    const uint32_t g = g0 + threadIdx.x / lanes;
    const uint32_t lo = g * a.cg > slab_c0 ? g * a.cg : slab_c0;
    const uint32_t hi = (g + 1) * a.cg < slab_c0 + width ? (g + 1) * a.cg : slab_c0 + width;
    float s = 0.0f, q = 0.0f;
    if (g < a.G) {
      for (uint32_t c = lo + lane; c < hi; c += lanes) {
        const float2 t = pair(c);
        s += t.x;
        q += t.y;
      }
    }
    for (uint32_t d = lanes / 2; d > 0; d >>= 1) {
      s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
      q += __shfl_xor_sync(0xFFFFFFFFu, q, d);
    }
    if (g < a.G && lane == 0) groups[g] = done(g, s, q);
  }
}
// Elements of group g in channels [c0, c0 + width) and the rows from row0 on, `most` of them at the most.
__device__ __forceinline__ float elements(const NormArgs& a, uint32_t g, uint32_t c0, uint32_t width, uint64_t row0, uint64_t most) {
  const uint32_t lo = g * a.cg > c0 ? g * a.cg : c0, hi = (g + 1) * a.cg < c0 + width ? (g + 1) * a.cg : c0 + width;
  const uint64_t left = a.L > row0 ? a.L - row0 : 0;
  return lo < hi ? (float)(hi - lo) * (float)(uint32_t)(left < most ? left : most) : 0.0f;      // L is under 2^31
}
// Those of part i of a sample (a cluster's): i counts the clusters of a slab first.  Every cluster's first block has rows, so 32 bits hold them.
__device__ __forceinline__ float elements_of_part(const NormArgs& a, uint32_t i, uint32_t g, uint32_t slab_width) {
  uint32_t channels = a.cg;
  if (a.slabs > 1) {
    const uint32_t clusters = a.chunks / kCluster, slab = i / clusters, c0 = slab * slab_width;
    const uint32_t lo = g * a.cg > c0 ? g * a.cg : c0, hi = (g + 1) * a.cg < c0 + slab_width ? (g + 1) * a.cg : c0 + slab_width;
    if (lo >= hi) return 0.0f;
    channels = hi - lo;
    i -= slab * clusters;
  }
  const uint32_t rows = a.rows_per_chunk * kCluster, left = (uint32_t)a.L - i * rows;
  return (float)channels * (float)(left < rows ? left : rows);
}

// The parts of a group joined by kLanes neighbouring threads, of which this is number k, kHeld parts a thread at a time: forward mean
// and sum of squares of the whole, backward the sums.  Eight threads hold the 64 parts that there can be without a launch between:
// read once, together (2 x 4096 x 640: 4.5 -> 2 us of the second launch).
template <bool kBackward, int kLanes, int kHeld>
__device__ __forceinline__ float2 join_parts(const NormArgs& a, uint32_t b, uint32_t g, uint32_t k) {
  const float2* in = a.partial + (size_t)b * a.parts * a.G + g;
  auto all = [](float v) {
#pragma unroll
    for (int d = 1; d < (kLanes < 32 ? kLanes : 32); d <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    if constexpr (kLanes == kThreads) {
      __shared__ float warps[kWarps];
      __syncthreads();
      if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
      __syncthreads();
      v = warps[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) v += warps[w];
    }
    return v;
  };
  const uint32_t parts = g < a.G ? a.parts : 0;
  const uint32_t slab_width = a.slabs == 1 ? a.C : a.slab_vecs * a.V;
  // a part that has elements of the group: the first of its first slab
  const float shift = !kBackward && parts ? in[(size_t)(a.slabs == 1 ? 0 : g * a.cg / slab_width * (a.chunks / kCluster)) * a.G].x : 0.0f;
  float2 t[kHeld];
  auto read = [&](uint32_t i0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const uint32_t i = i0 + j * kLanes;
      t[j] = i < parts ? in[(size_t)i * a.G] : make_float2(0.0f, 0.0f);
    }
  };
  auto elements_at = [&](uint32_t i) { return i < parts ? elements_of_part(a, i, g, slab_width) : 0.0f; };
  float s = 0.0f, q = 0.0f;
  for (uint32_t i0 = k; i0 < parts; i0 += kHeld * kLanes) {
    read(i0);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (kBackward) {
        s += t[j].x;
        q += t[j].y;
      } else {
        const float n = elements_at(i0 + j * kLanes);
        if (n > 0.0f) s += n * (t[j].x - shift);
      }
    }
  }
  s = all(s);
  if (kBackward) return make_float2(s, all(q));
  const float mean = shift + s / ((float)a.L * (float)a.cg);
  for (uint32_t i0 = k; i0 < parts; i0 += kHeld * kLanes) {
    if (kLanes == kThreads) read(i0);      // eight threads hold them all
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const float n = elements_at(i0 + j * kLanes);
      if (n > 0.0f) q += fmaf(n * (t[j].x - mean), t[j].x - mean, t[j].y);
    }
  }
  return make_float2(mean, all(q));
}

// Launches.  A call's first kernel is launched in the ordinary way: it starts when everything ahead of the call is complete, and its writes
// visible.  The others are programmatic launches: the second kernel starts when all blocks of the first have, so it may read the call's
// inputs at once.  It sends its first rows on their way, past L1, while the first kernel ends, and waits before it reads anything else or
// writes.  (With a programmatic first launch too, the second would read inputs that only the first has waited for.)
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <int V>
__global__ void __launch_bounds__(kThreads, 4) group_stats_kernel(const __grid_constant__ NormArgs a) {
  launch_next();
  extern __shared__ uint4 ring[];
  float2* sh = sums_of<V>(ring);
  const Place<V> p(a);
  const __nv_bfloat16* xs = a.x + (size_t)p.b * a.L * a.C;
  const __nv_bfloat16* const src[1] = {xs + (p.row0 + p.lane_row) * a.C + p.c0};
  Walk<1, V, false> way(src, p.live ? p.rows : 0, p.lane_row, p.row_step, a.C, ring);
  const __nv_bfloat16* first_row = xs + (p.rows ? p.row0 : 0) * a.C;      // the chunk's
  const uint32_t slab_c0 = p.slab * a.slab_vecs * V;
  const uint32_t width = a.C - slab_c0 < a.slab_vecs * V ? a.C - slab_c0 : a.slab_vecs * V;
  float2* groups = sh + kThreads * V;
  float* shifts = reinterpret_cast<float*>(groups + a.G);
  const uint32_t g_end = (slab_c0 + width - 1) / a.cg + 1;
  for (uint32_t g = slab_c0 / a.cg + threadIdx.x; g < g_end; g += kThreads) {
    const __nv_bfloat16* at = first_row + g * a.cg;
    const uint32_t last = p.rows ? p.rows - 1 : 0;
    const float u = __bfloat162float(*at), v = __bfloat162float(at[(size_t)(last / 2) * a.C]), w = __bfloat162float(at[(size_t)last * a.C]);
    shifts[g] = fmaxf(fminf(u, v), fminf(fmaxf(u, v), w));
  }
  __syncthreads();
  F2 shift[kPairs<V>], s[kPairs<V>], q[kPairs<V>];      // the shift's negative
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    s[i] = q[i] = F2(0.0f, 0.0f);
    float2 t = make_float2(0.0f, 0.0f);
    if (p.live) {
      t.x = -shifts[group_of(p.c0 + 2 * i, a.by_cg)];
      if (V > 1) t.y = -shifts[group_of(p.c0 + 2 * i + 1, a.by_cg)];
    }
    shift[i] = F2(t.x, t.y);
  }
  way.run([&](ptrdiff_t, const Vec<V>(&v)[1]) {
    F2 f[kPairs<V>];
    unpack<V>(v[0], f);
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      const F2 d = add(f[i], shift[i]);
      s[i] = add(s[i], d);
      q[i] = fma(d, d, q[i]);
    }
  });
  join_rows<V>(p, s, q, sh, width);
  join_channels(a, slab_c0, width, groups, [&](uint32_t c) { return sh[place_of<V>(c - slab_c0, width)]; }, [&](uint32_t g, float sum, float sum2) {
    const float n = elements(a, g, slab_c0, width, p.row0, p.rows);
    if (n == 0.0f) return make_float2(0.0f, 0.0f);
    const float off = sum / n;
    // fmaxf would turn the NaN of a NaN or an infinity into 0
    return make_float2(shifts[g] + off, sum2 < INFINITY ? fmaxf(sum2 - sum * off, 0.0f) : NAN);
  });
  cluster_sync_all();
  // mean and sum of squares of the cluster's blocks, joined
  join_cluster(groups, a.G, a.partial + ((size_t)p.b * a.parts + p.slab * (a.chunks / kCluster) + p.chunk / kCluster) * a.G, [](uint32_t i) { return i; },
               [&](uint32_t g, const float2 (&v)[kCluster]) {
    const uint64_t row0 = (uint64_t)(p.chunk / kCluster * kCluster) * a.rows_per_chunk;
    float n[kCluster], total = 0.0f, mean = 0.0f, m2 = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kCluster; ++k) {
      n[k] = elements(a, g, slab_c0, width, row0 + (uint64_t)k * a.rows_per_chunk, a.rows_per_chunk);
      total += n[k];
    }
    if (total == 0.0f) return make_float2(0.0f, 0.0f);
#pragma unroll
    for (uint32_t k = 1; k < kCluster; ++k) mean += n[k] > 0.0f ? n[k] * (v[k].x - v[0].x) : 0.0f;      // block 0 has rows where any has
    mean = v[0].x + mean / total;
#pragma unroll
    for (uint32_t k = 0; k < kCluster; ++k) m2 += n[k] > 0.0f ? fmaf(n[k] * (v[k].x - mean), v[k].x - mean, v[k].y) : 0.0f;
    return make_float2(mean, m2);
  });
  cluster_sync_all();
}

// What the second launch needs of a group: mean and rstd, or backward the means of s1 and s2.
template <bool kBackward>
__device__ __forceinline__ float2 finish(const NormArgs& a, float2 t) {
  const float inv_n = 1.0f / ((float)a.L * (float)a.cg);
  if (kBackward) return make_float2(t.x * inv_n, t.y * inv_n);
  return make_float2(t.x, rsqrtf(t.y * inv_n + a.eps));
}
template <bool kBackward>
__device__ __forceinline__ void finish_all(const NormArgs& a, uint32_t b, float2* out) {
  if (a.finished) {
    for (uint32_t g = threadIdx.x; g < a.G; g += kThreads) out[g] = a.finished[(size_t)b * a.G + g];
  } else {
    for (uint32_t g0 = 0; g0 < a.G; g0 += kThreads / 8) {      // eight threads a group
      const uint32_t g = g0 + threadIdx.x / 8;
      const float2 t = join_parts<kBackward, 8, kMostParts / 8>(a, b, g, threadIdx.x % 8);
      if (g < a.G && threadIdx.x % 8 == 0) out[g] = finish<kBackward>(a, t);
    }
  }
  __syncthreads();
}
// A block for each group of sample blockIdx.y.  (A warp for each took 19 us at 592 parts, waiting for one load after another.)
template <bool kBackward>
__global__ void __launch_bounds__(kThreads) group_finish_kernel(const __grid_constant__ NormArgs a) {
  pdl_prologue();
  const uint32_t g = blockIdx.x, b = blockIdx.y;
  const float2 t = join_parts<kBackward, kThreads, 1>(a, b, g, threadIdx.x);
  if (threadIdx.x == 0) a.finished[(size_t)b * a.G + g] = finish<kBackward>(a, t);
}

// Codes of eight channels a thread.  16 neighbouring lanes hold a block of 128 channels of a row (C / 8 and a slab's width are multiples
// of 16) and have the same rows; the other half of the warp may have one more.
__device__ __forceinline__ uint2 encode_row_block(const uint4& raw, float& scale) {
  uint32_t m = max_abs2(max_abs2(raw.x, raw.y), max_abs2(raw.z, raw.w));
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) m = max_abs2(m, __shfl_xor_sync(0xFFFFu << (threadIdx.x & 16), m, d));
  scale = fp8_scale_of(larger_of(m));
  float y[8];
  unpack8(raw, y);
  return fp8_encode8(y, scale, fp8_factor_of(scale));
}

// Weight and bias of a thread's channels, and (with) whatever f makes of the weight and the group's statistics of each.
template <int V>
struct Params {
  float w[2 * kPairs<V>] = {}, b[2 * kPairs<V>] = {};
  __device__ __forceinline__ Params(const NormArgs& a, const Place<V>& p) {
    if (!p.live) return;
    params<V>(a.weight, a.params_f32, p.c0, 1.0f, reinterpret_cast<float(&)[V]>(w));
    params<V>(a.bias, a.params_f32, p.c0, 0.0f, reinterpret_cast<float(&)[V]>(b));
  }
  template <typename F>
  __device__ __forceinline__ void with(const NormArgs& a, const Place<V>& p, const float2* stats, F&& f, F2 (&bias)[kPairs<V>], F2 (&u)[kPairs<V>], F2 (&v)[kPairs<V>]) const {
    float fu[2 * kPairs<V>] = {}, fv[2 * kPairs<V>] = {};
    if (p.live) {
#pragma unroll
      for (int i = 0; i < V; ++i) f(w[i], stats[group_of(p.c0 + i, a.by_cg)], fu[i], fv[i]);
    }
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      bias[i] = F2(b[2 * i], b[2 * i + 1]);
      u[i] = F2(fu[2 * i], fu[2 * i + 1]);
      v[i] = F2(fv[2 * i], fv[2 * i + 1]);
    }
  }
};

template <int V, bool kCodes>
__global__ void __launch_bounds__(kThreads, 4) group_apply_kernel(const __grid_constant__ NormArgs a) {
  launch_next();
  extern __shared__ uint4 ring[];
  float2* sh = sums_of<V>(ring);
  const Place<V> p(a, true);
  // From the chunk's end to its start: what the first launch read last is still in L2.
  const size_t first = ((size_t)p.b * a.L + p.row0 + p.lane_row) * a.C + p.c0;
  const __nv_bfloat16* const src[1] = {a.x + first};
  Walk<1, V, true> way(src, p.live ? p.rows : 0, p.lane_row, p.row_step, a.C, ring);
  wait_for_earlier();
  finish_all<false>(a, p.b, sh);
  const Params<V> params(a, p);
  if (p.chunk == 0 && p.slab == 0 && a.finished == nullptr)
    for (uint32_t g = threadIdx.x; g < a.G; g += kThreads) reinterpret_cast<float2*>(a.stats)[(size_t)p.b * a.G + g] = sh[g];
  F2 mean[kPairs<V>], scale[kPairs<V>], bias[kPairs<V>];      // the mean's negative
  params.with(a, p, sh, [](float w, float2 t, float& m, float& s) { m = -t.x; s = t.y * w; }, bias, mean, scale);
  way.run([&](ptrdiff_t at, const Vec<V>(&v)[1]) {
    F2 f[kPairs<V>];
    unpack<V>(v[0], f);
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      const F2 h = fma(add(f[i], mean[i]), scale[i], bias[i]);      // first the difference: a group of equal values gives exactly the bias
      f[i] = a.silu ? mul(h, sigmoid(h)) : h;
    }
    store<V>(a.y + first + at, f, a.stream);
    if constexpr (kCodes) {
      // the codes are those of the BF16 output
      float s;
      *reinterpret_cast<uint2*>(a.codes + first + at) = encode_row_block(make_uint4(to_bf16x2(f[0]), to_bf16x2(f[1]), to_bf16x2(f[2]), to_bf16x2(f[3])), s);
      if ((p.vec & 15) == 0) a.code_scales[(first + at) / 128] = s;
    }
  });
}

// dy * act'(h)
__device__ __forceinline__ F2 grad_h(F2 h, F2 dy, int silu) {
  if (!silu) return dy;
  const F2 g = sigmoid(h), one(1.0f, 1.0f), minus(-1.0f, -1.0f);
  return mul(dy, mul(g, fma(h, fma(g, minus, one), one)));
}

template <int V>
__global__ void __launch_bounds__(kThreads, 3) group_grad_sums_kernel(const __grid_constant__ NormArgs a) {
  launch_next();
  extern __shared__ uint4 ring[];
  float2* sh = sums_of<V>(ring);
  const Place<V> p(a);
  const float2* stats = reinterpret_cast<const float2*>(a.stats) + (size_t)p.b * a.G;
  const size_t first = ((size_t)p.b * a.L + p.row0 + p.lane_row) * a.C + p.c0;
  const __nv_bfloat16* const src[2] = {a.x + first, a.dy + first};
  Walk<2, V, false> way(src, p.live ? p.rows : 0, p.lane_row, p.row_step, a.C, ring);
  F2 mean[kPairs<V>], scale[kPairs<V>], bias[kPairs<V>], s[kPairs<V>], q[kPairs<V>];      // the mean's negative
  Params<V>(a, p).with(a, p, stats, [](float w, float2 t, float& m, float& sc) { m = -t.x; sc = t.y * w; }, bias, mean, scale);
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) s[i] = q[i] = F2(0.0f, 0.0f);
  way.run([&](ptrdiff_t, const Vec<V>(&v)[2]) {
    F2 x[kPairs<V>], dy[kPairs<V>];
    unpack<V>(v[0], x);
    unpack<V>(v[1], dy);
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      const F2 d = add(x[i], mean[i]), dh = grad_h(fma(d, scale[i], bias[i]), dy[i], a.silu);
      s[i] = add(s[i], dh);
      q[i] = fma(dh, d, q[i]);      // times rstd at the end
    }
  });
  if (p.live) {
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i)
      q[i] = mul(q[i], F2(stats[group_of(p.c0 + 2 * i, a.by_cg)].y, V > 1 ? stats[group_of(p.c0 + 2 * i + 1, a.by_cg)].y : 0.0f));
  }
  const uint32_t slab_c0 = p.slab * a.slab_vecs * V;
  const uint32_t width = a.C - slab_c0 < a.slab_vecs * V ? a.C - slab_c0 : a.slab_vecs * V;
  join_rows<V>(p, s, q, sh, width);
  float2* groups = sh + kThreads * V;
  join_channels(a, slab_c0, width, groups, [&](uint32_t c) {
    const float w = param(a.weight, a.params_f32, c, 1.0f);
    const float2 t = sh[place_of<V>(c - slab_c0, width)];
    return make_float2(w * t.x, w * t.y);
  }, [](uint32_t, float sum, float sum2) { return make_float2(sum, sum2); });
  const uint32_t part = p.chunk / kCluster;
  cluster_sync_all();
  join_cluster(groups, a.G, a.partial + ((size_t)p.b * a.parts + p.slab * (a.chunks / kCluster) + part) * a.G, [](uint32_t i) { return i; },
               [](uint32_t, const float2 (&v)[kCluster]) { return add_up(v); });
  join_cluster(sh, width, a.channel_partial + ((size_t)p.b * (a.chunks / kCluster) + part) * a.C + slab_c0, [&](uint32_t c) { return place_of<V>(c, width); },
               [](uint32_t, const float2 (&v)[kCluster]) { return add_up(v); });
  cluster_sync_all();
}

// The blocks of one more sample than there are add the channel sums up to dweight and dbias.
template <int V>
__global__ void __launch_bounds__(kThreads, 3) group_grad_apply_kernel(const __grid_constant__ NormArgs a) {
  launch_next();
  extern __shared__ uint4 ring[];
  float2* sh = sums_of<V>(ring);
  if (blockIdx.z == a.B) {
    wait_for_earlier();
    // a warp's 32 lanes take 32 neighbouring channels, the eight warps every eighth part
    __shared__ float2 part[kWarps][32];
    const uint32_t lane = threadIdx.x & 31, wp = threadIdx.x >> 5, parts = a.B * (a.chunks / kCluster);
    for (uint32_t c0 = (blockIdx.y * gridDim.x + blockIdx.x) * 32; c0 < a.C; c0 += gridDim.x * gridDim.y * 32) {
      const uint32_t c = c0 + lane;
      float2 t = make_float2(0.0f, 0.0f);
      if (c < a.C) {
#pragma unroll 4
        for (uint32_t i = wp; i < parts; i += kWarps) {
          const float2 u = a.channel_partial[(size_t)i * a.C + c];
          t.x += u.x;
          t.y += u.y;
        }
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
      __syncthreads();
    }
    return;
  }
  const Place<V> p(a, true);
  const size_t first = ((size_t)p.b * a.L + p.row0 + p.lane_row) * a.C + p.c0;
  const __nv_bfloat16* const src[2] = {a.x + first, a.dy + first};
  Walk<2, V, true> way(src, p.live ? p.rows : 0, p.lane_row, p.row_step, a.C, ring);      // from the chunk's end, as in the forward pass
  wait_for_earlier();
  const Params<V> params(a, p);
  finish_all<true>(a, p.b, sh);
  // dx = scale * dh - rstd^2 * m2 * (x - mean) - rstd * m1; h = (x - mean) * scale + bias.  First the difference, as in the passes before:
  // in a group of equal values far from zero a factor and an offset of x would each be large, and h off by what their sum rounds away.
  const float2* stats = reinterpret_cast<const float2*>(a.stats) + (size_t)p.b * a.G;
  F2 scale[kPairs<V>], bias[kPairs<V>], slope[kPairs<V>], rest[kPairs<V>], mean[kPairs<V>];      // the mean's negative
  params.with(a, p, stats, [](float w, float2 t, float& m, float& sc) { m = -t.x; sc = t.y * w; }, bias, mean, scale);
  if (!p.live) return;
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    float sl[2] = {}, re[2] = {};
#pragma unroll
    for (int k = 0; k < 2 && 2 * i + k < V; ++k) {
      const uint32_t g = group_of(p.c0 + 2 * i + k, a.by_cg);
      const float2 t = stats[g], m = sh[g];
      sl[k] = -t.y * t.y * m.y;
      re[k] = -t.y * m.x;
    }
    slope[i] = F2(sl[0], sl[1]);
    rest[i] = F2(re[0], re[1]);
  }
  way.run([&](ptrdiff_t at, const Vec<V>(&v)[2]) {
    F2 x[kPairs<V>], dy[kPairs<V>];
    unpack<V>(v[0], x);
    unpack<V>(v[1], dy);
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      const F2 d = add(x[i], mean[i]), dh = grad_h(fma(d, scale[i], bias[i]), dy[i], a.silu);
      x[i] = fma(scale[i], dh, fma(slope[i], d, rest[i]));
    }
    store<V>(a.y + first + at, x, a.stream);
  });
}

int sm_count_here() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// How a call is cut: the width of a thread's channel vector, slabs of channels, chunks of positions.
struct Plan {
  int V;
  uint32_t slab_vecs, slabs, chunks, parts;
  uint64_t rows_per_chunk;
};
Plan plan(uint32_t B, uint64_t L, uint32_t C, bool aligned16, bool aligned4, bool backward, int sms) {
  Plan p;
  p.V = (C % 8 == 0 && aligned16) ? 8 : (C % 2 == 0 && aligned4) ? 2 : 1;
  const uint32_t nvec = C / p.V;
  // The width of a slab: the one that leaves the fewest threads without a channel, at 1280 channels 80 vectors (three rows in 256
  // threads) and not 160 (one).  With slabs it is a multiple of 16 vectors: a block of 128 channels lies in one of them.
  uint32_t best = 0;
  for (uint32_t slabs = (nvec + kThreads - 1) / kThreads, k = 0; k < 4; ++slabs, ++k) {
    const uint32_t even = (nvec + slabs - 1) / slabs, width = slabs == 1 ? even : (even + 15) / 16 * 16;
    if (width > kThreads || (k > 0 && width < 64)) continue;      // 1024 neighbouring bytes at least
    const uint32_t count = (nvec + width - 1) / width, used = nvec * (kThreads / width) * 1024 / (count * kThreads);   // of 1024
    if (used > best + 64 * (best > 0)) { best = used; p.slabs = count; p.slab_vecs = width; }
  }
  // All the thread blocks that fit on the SMs at a time, with eight rows a thread at least.  Where each would have over 64, three times
  // as many: SMs differ in speed, and with one block for each place the slowest is waited for (1024 x 1024 x 128).
  const uint64_t places = (uint64_t)sms * (backward ? 3 : 4), samples = (uint64_t)B * p.slabs;
  uint64_t want = places / samples > 1 ? places / samples : 1;
  const uint32_t row_step = kThreads / p.slab_vecs;
  if (L / (want * row_step) > 64) want = 3 * places / samples > 1 ? 3 * places / samples : 1;
  const uint64_t most = (L + (uint64_t)row_step * 8 - 1) / ((uint64_t)row_step * 8);
  uint64_t chunks = want < most ? want : most;
  if (chunks > 4096) chunks = 4096;
  chunks = chunks < kCluster ? kCluster : chunks / kCluster * kCluster;
  p.rows_per_chunk = (L + chunks - 1) / chunks;
  chunks = (L + p.rows_per_chunk - 1) / p.rows_per_chunk;
  p.chunks = (uint32_t)((chunks + kCluster - 1) / kCluster * kCluster);
  p.parts = p.chunks / kCluster * p.slabs;
  return p;
}
bool finishes(const Plan& p) { return p.parts > kMostParts; }
size_t group_pairs(const Plan& p, uint32_t B, uint32_t G) { return ((size_t)B * p.parts * G + 1) / 2 * 2; }   // whole 16 bytes
size_t partial_pairs(const Plan& p, uint32_t B, uint32_t C, uint32_t G, bool backward) {
  return group_pairs(p, B, G) + (backward ? (size_t)B * (p.chunks / kCluster) * C : 0) + (finishes(p) && backward ? (size_t)B * G : 0);
}
bool al(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check(const char* who, uint64_t B, uint64_t L, uint64_t C, uint64_t G, int activation, int param_dtype) {
  const char* what = nullptr;
  if (G == 0 || C == 0 || C % G != 0) what = "the channels must be a positive multiple of the groups";
  else if (C > 65536) what = "at most 65536 channels";
  else if (G > kMostGroups) what = "at most 4096 groups";
  else if (B > 65534 || L > 0x7FFFFFFFull) what = "at most 65534 samples of at most 2^31 - 1 positions";
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

// first: of a call, in clusters, and behind all that is ahead in the stream
template <auto kKernel>
cudaError_t launch(dim3 grid, bool first, size_t smem, cudaStream_t stream, const NormArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  int n = 0;
  if (first) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = kCluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (!first && pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (smem > 46 * 1024) {      // beside two kilobytes that are not dynamic
    static std::atomic<uint64_t> allowed{0};     // a bit for each device on which the kernel may use this much
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev)) return e;
    if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
      if (const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared)) return e;
      if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
  }
  return cudaLaunchKernelEx(&cfg, kKernel, a);
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
    const size_t f = partial_pairs(plan((uint32_t)B, L, (uint32_t)C, k == 0, k <= 1, backward != 0, sm_count_here()), (uint32_t)B, (uint32_t)C, (uint32_t)G, backward != 0);
    most = f > most ? f : most;
  }
  return most * sizeof(float2);
}

int flame_group_norm(const void* x, const void* weight, const void* bias, void* y, void* codes, void* code_scales, void* stats,
                     size_t B, size_t L, size_t C, size_t G, float eps, int activation, int param_dtype, void* workspace,
                     size_t workspace_bytes, void* stream) {
  const char* who = "flame_group_norm";
  if (const int e = check(who, B, L, C, G, activation, param_dtype)) return e;
  if (B == 0 || L == 0) return 0;
  if (!x || !y || !stats || !workspace) return refuse(who, "null tensor");
  if (workspace_bytes < flame_group_norm_workspace_bytes(B, L, C, G, 0)) return refuse(who, "workspace too small");
  const uintptr_t psize = param_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2;
  if (!al(x, 2) || !al(y, 2) || !al(weight, psize) || !al(bias, psize) || !al(stats, 8) || !al(code_scales, 4) || !al(workspace, 16))
    return refuse(who, "misaligned tensor (stats: 8 bytes)");
  const bool al16 = al(x, 16) && al(y, 16);
  if (codes && (C % 128 != 0 || !al16 || !al(codes, 8) || !code_scales)) return refuse(who, "codes need channels % 128 == 0, 16-byte aligned tensors and a place for the scales");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  const Plan p = plan((uint32_t)B, L, (uint32_t)C, al16, al(x, 4) && al(y, 4), false, sm_count_here());
  NormArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.weight = weight; a.bias = bias; a.y = static_cast<__nv_bfloat16*>(y);
  a.codes = static_cast<uint8_t*>(codes); a.code_scales = static_cast<float*>(code_scales); a.stats = static_cast<float*>(stats);
  a.partial = static_cast<float2*>(workspace);
  if (finishes(p)) a.finished = reinterpret_cast<float2*>(a.stats);
  a.B = (uint32_t)B; a.C = (uint32_t)C; a.G = (uint32_t)G; a.cg = (uint32_t)(C / G); a.L = L;
  a.by_cg = a.cg == 1 ? 0 : (uint32_t)(((1ull << 32) + a.cg - 1) / a.cg);
  a.chunks = p.chunks; a.parts = p.parts; a.rows_per_chunk = (uint32_t)p.rows_per_chunk; a.slabs = p.slabs; a.slab_vecs = p.slab_vecs; a.V = (uint32_t)p.V;
  a.eps = eps; a.silu = activation == FLAME_ACTIVATION_SILU; a.stream = B * L * C > (24u << 20); a.params_f32 = param_dtype == FLAME_OFFLOAD_DTYPE_F32;
  const dim3 grid(p.chunks, p.slabs, (unsigned)B);
  const size_t ring = p.V == 8 ? kRingBytes : 0, sums = ring + ((size_t)kThreads * p.V + G) * sizeof(float2), groups = ring + G * sizeof(float2);
  const size_t sums_and_shifts = sums + G * sizeof(float);
  cudaStream_t s = (cudaStream_t)stream;
  return cuda_result(who, by_width(p.V, [&](auto v) {
    constexpr int V = decltype(v)::value;
    cudaError_t e = launch<group_stats_kernel<V>>(grid, true, sums_and_shifts, s, a);
    if (e != cudaSuccess) return e;
    if (a.finished) e = launch<group_finish_kernel<false>>(dim3(a.G, a.B), false, 0, s, a);
    if (e != cudaSuccess) return e;
    if constexpr (V == 8) {
      if (a.codes) return launch<group_apply_kernel<8, true>>(grid, false, groups, s, a);
    }
    return launch<group_apply_kernel<V, false>>(grid, false, groups, s, a);
  }));
}

int flame_group_norm_backward(const void* x, const void* dy, const void* weight, const void* bias, const void* stats, void* dx,
                              void* dweight, void* dbias, size_t B, size_t L, size_t C, size_t G, int activation, int param_dtype,
                              void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "flame_group_norm_backward";
  if (const int e = check(who, B, L, C, G, activation, param_dtype)) return e;
  cudaStream_t s = (cudaStream_t)stream;
  const size_t psize = param_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2;
  if (B == 0 || L == 0) {   // sums over nothing
    if (dweight) if (const cudaError_t e = cudaMemsetAsync(dweight, 0, C * psize, s)) return cuda_result(who, e);
    if (dbias) if (const cudaError_t e = cudaMemsetAsync(dbias, 0, C * psize, s)) return cuda_result(who, e);
    return 0;
  }
  if (!x || !dy || !dx || !stats || !workspace) return refuse(who, "null tensor");
  if (workspace_bytes < flame_group_norm_workspace_bytes(B, L, C, G, 1)) return refuse(who, "workspace too small");
  if (!al(x, 2) || !al(dy, 2) || !al(dx, 2) || !al(weight, psize) || !al(bias, psize) || !al(dweight, psize) || !al(dbias, psize) || !al(stats, 8) || !al(workspace, 16))
    return refuse(who, "misaligned tensor (stats: 8 bytes)");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  const Plan p = plan((uint32_t)B, L, (uint32_t)C, al(x, 16) && al(dy, 16) && al(dx, 16), al(x, 4) && al(dy, 4) && al(dx, 4), true, sm_count_here());
  NormArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.dy = static_cast<const __nv_bfloat16*>(dy); a.weight = weight; a.bias = bias;
  a.y = static_cast<__nv_bfloat16*>(dx); a.stats = const_cast<float*>(static_cast<const float*>(stats));
  a.partial = static_cast<float2*>(workspace);
  a.channel_partial = a.partial + group_pairs(p, (uint32_t)B, (uint32_t)G);
  if (finishes(p)) a.finished = a.channel_partial + (size_t)B * (p.chunks / kCluster) * C;
  a.dweight = dweight; a.dbias = dbias;
  a.B = (uint32_t)B; a.C = (uint32_t)C; a.G = (uint32_t)G; a.cg = (uint32_t)(C / G); a.L = L;
  a.by_cg = a.cg == 1 ? 0 : (uint32_t)(((1ull << 32) + a.cg - 1) / a.cg);
  a.chunks = p.chunks; a.parts = p.parts; a.rows_per_chunk = (uint32_t)p.rows_per_chunk; a.slabs = p.slabs; a.slab_vecs = p.slab_vecs; a.V = (uint32_t)p.V;
  a.silu = activation == FLAME_ACTIVATION_SILU; a.stream = B * L * C > (24u << 20); a.params_f32 = param_dtype == FLAME_OFFLOAD_DTYPE_F32;
  const dim3 grid(p.chunks, p.slabs, (unsigned)B);
  const dim3 more(p.chunks, p.slabs, (unsigned)B + (dweight || dbias ? 1 : 0));
  const size_t ring = p.V == 8 ? kRingBytes : 0, sums = ring + ((size_t)kThreads * p.V + G) * sizeof(float2), groups = ring + G * sizeof(float2);
  return cuda_result(who, by_width(p.V, [&](auto v) {
    constexpr int V = decltype(v)::value;
    cudaError_t e = launch<group_grad_sums_kernel<V>>(grid, true, sums, s, a);
    if (e != cudaSuccess) return e;
    if (a.finished) e = launch<group_finish_kernel<true>>(dim3(a.G, a.B), false, 0, s, a);
    if (e != cudaSuccess) return e;
    return launch<group_grad_apply_kernel<V>>(more, false, groups, s, a);
  }));
}

}  // extern "C"
