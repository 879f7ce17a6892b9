// Matrix product of FP8 E4M3 operands with one fp32 scale for each block of 128, written for sm_100a, and the quantiser that
// makes such operands from BF16 matrices.
//
//   C[m][n] = sum over blocks kb of sa(m, kb) * sb(n, kb) * (sum over k in kb of a(m, k) * b(n, k))
//
// A block runs along the contraction: 1 x 128 of a row ("rows"), 128 x 1 of a column ("columns"), or 128 x 128 ("tiles", a
// weight, which then serves the product and its transpose with the same codes).
//
// Times in this file: calls recorded in a CUDA graph and replayed back to back on one B200, a few milliseconds at a time, so that the
// board's power limit is not reached unless it says so.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "codec_kernels.cuh"
#include "common.h"
#include "fp8_device.cuh"

namespace flame_b200 {
namespace {

constexpr int kBlock = 128;

// ---- quantiser ------------------------------------------------------------------
// A thread block owns a 128 x 128 tile: thread (r, c) = (t / 16, t % 16) holds columns 8c..8c+7 of rows r, r + 16, ..., r + 112
// as eight 16-byte loads, and keeps them in registers for whichever scales the caller wants: of its rows (four shuffles), of its
// columns (one shuffle and eight partial maxima through shared memory), or of the tile.  The source is read once for both.  Bound by
// memory with one kind of scales (8192 x 8192 rows 33.5 us, tiles 33.1: 6.0 TB/s), by instructions with two (rows and columns 51.7 us,
// 5.2 TB/s).  Rows that are no multiple of 16 bytes apart are read element by element (1000 x 1331 6.3 us, 1000 x 1328 3.3).
constexpr int kQuantThreads = 256;

enum : uint32_t { kQuantRows = 1, kQuantTiles = 2, kQuantColumns = 4, kQuantWide = 8 };   // kQuantWide: 16-byte loads are possible

struct QuantJob {
  const __nv_bfloat16* x;
  size_t x_stride;
  uint32_t rows, cols;
  uint8_t* row_codes;        // rows or tiles
  float* row_scales;
  uint8_t* col_codes;        // columns
  float* col_scales;
  size_t code_stride;
  uint32_t tiles_across;     // ceil(cols / 128)
  uint32_t tiles;
  uint32_t mode;
};
// Up to three matrices in a launch: a layer's output gradient, input and weight.
struct QuantJobs { QuantJob job[3]; };

__global__ void __launch_bounds__(kQuantThreads, 4) fp8_quant_kernel(const __grid_constant__ QuantJobs jobs) {
  pdl_prologue();
  __shared__ uint32_t part[8][kBlock / 2];       // packed maxima of two columns
  __shared__ __align__(16) float factors[kBlock];
  __shared__ __align__(16) float scales[kBlock];
  uint32_t tile = blockIdx.x, which = 0;
  while (which < 2 && tile >= jobs.job[which].tiles) tile -= jobs.job[which++].tiles;
  const QuantJob& a = jobs.job[which];
  const uint32_t tm = tile / a.tiles_across, tn = tile - tm * a.tiles_across;
  const uint32_t t = threadIdx.x, lr = t >> 4, lc = t & 15;
  const uint32_t row0 = tm * kBlock + lr, col = tn * kBlock + lc * 8;
  uint4 raw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) raw[j] = make_uint4(0u, 0u, 0u, 0u);
  if (col < a.cols) {
    const __nv_bfloat16* src = a.x + (size_t)row0 * a.x_stride + col;
    if (a.mode & kQuantWide) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (row0 + 16 * j < a.rows) raw[j] = __ldcs(reinterpret_cast<const uint4*>(src + (size_t)(16 * j) * a.x_stride));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (row0 + 16 * j < a.rows) {
          uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (col + i < a.cols) w[i / 2] |= (uint32_t)__bfloat16_as_ushort(src[(size_t)(16 * j) * a.x_stride + i]) << (16 * (i & 1));
          raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
  }
  auto put = [&](uint8_t* codes, int j, const uint2& c) {      // a row's padding gets zeros
    if (row0 + 16 * j < a.rows && col < a.cols) *reinterpret_cast<uint2*>(codes + (size_t)(row0 + 16 * j) * a.code_stride + col) = c;
  };
  if (a.mode & kQuantRows) {
    // 16 lanes hold a row.  Each lane takes the maximum of one of its eight rows to a scale and a factor, and the others ask it.
    float mine = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t m = max_abs2(max_abs2(raw[j].x, raw[j].y), max_abs2(raw[j].z, raw[j].w));
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) m = max_abs2(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
      if ((lc & 7) == (uint32_t)j) mine = larger_of(m);
    }
    const float scale = fp8_scale_of(mine), factor = fp8_factor_of(scale);
    if (lc < 8 && row0 + 16 * lc < a.rows) a.row_scales[(size_t)(row0 + 16 * lc) * a.tiles_across + tn] = scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float fj = __shfl_sync(0xFFFFFFFFu, factor, j, 16), sj = __shfl_sync(0xFFFFFFFFu, scale, j, 16);
      float f[8];
      unpack8(raw[j], f);
      put(a.row_codes, j, fp8_encode8(f, sj, fj));
    }
  }
  if (a.mode & (kQuantTiles | kQuantColumns)) {
    uint32_t c[4] = {0u, 0u, 0u, 0u};     // packed maxima of this thread's eight columns over its eight rows, and its neighbour's
#pragma unroll
    for (int j = 0; j < 8; ++j) { c[0] = max_abs2(c[0], raw[j].x); c[1] = max_abs2(c[1], raw[j].y); c[2] = max_abs2(c[2], raw[j].z); c[3] = max_abs2(c[3], raw[j].w); }
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = max_abs2(c[i], __shfl_xor_sync(0xFFFFFFFFu, c[i], 16));
    if ((t & 16) == 0) *reinterpret_cast<uint4*>(&part[t >> 5][lc * 4]) = make_uint4(c[0], c[1], c[2], c[3]);
    __syncthreads();
    if (t < 32) {      // a lane joins four columns
      uint32_t u = part[0][2 * t], v = part[0][2 * t + 1];
#pragma unroll
      for (int k = 1; k < 8; ++k) { u = max_abs2(u, part[k][2 * t]); v = max_abs2(v, part[k][2 * t + 1]); }
      float m[4];
      if (a.mode & kQuantTiles) {
        uint32_t w = max_abs2(u, v);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) w = max_abs2(w, __shfl_xor_sync(0xFFFFFFFFu, w, d));
        m[0] = m[1] = m[2] = m[3] = larger_of(w);
      } else {
        m[0] = fmaxf(__uint_as_float((u << 16) & 0x7FFF0000u), 0.0f);      // NaN counts as zero
        m[1] = fmaxf(__uint_as_float(u & 0x7FFF0000u), 0.0f);
        m[2] = fmaxf(__uint_as_float((v << 16) & 0x7FFF0000u), 0.0f);
        m[3] = fmaxf(__uint_as_float(v & 0x7FFF0000u), 0.0f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { scales[4 * t + i] = fp8_scale_of(m[i]); factors[4 * t + i] = fp8_factor_of(scales[4 * t + i]); }
    }
    __syncthreads();
    if (a.mode & kQuantTiles) {
      const float scale = scales[0], factor = factors[0];
      if (t == 0) a.row_scales[(size_t)tm * a.tiles_across + tn] = scale;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float f[8];
        unpack8(raw[j], f);
        put(a.row_codes, j, fp8_encode8(f, scale, factor));
      }
    } else {
      if (t < kBlock && tn * kBlock + t < a.cols) a.col_scales[(size_t)tm * a.cols + tn * kBlock + t] = scales[t];
      const float4 f0 = *reinterpret_cast<const float4*>(factors + lc * 8), f1 = *reinterpret_cast<const float4*>(factors + lc * 8 + 4);
      const float fc[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
      const uint64_t pc[4] = {fp8_factors(f0.x, f0.y), fp8_factors(f0.z, f0.w), fp8_factors(f1.x, f1.y), fp8_factors(f1.z, f1.w)};
      bool divides = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) divides |= fp8_divides(fc[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float f[8];
        unpack8(raw[j], f);
        if (divides) {
#pragma unroll 1
          for (int i = 0; i < 8; ++i) f[i] = fp8_divides(factors[lc * 8 + i]) ? __fdiv_rn(f[i], scales[lc * 8 + i]) : __fmul_rn(f[i], factors[lc * 8 + i]);
          put(a.col_codes, j, fp8_pack8(f));
        } else {
          put(a.col_codes, j, make_uint2(fp8_encode2(f[0], f[1], pc[0]) | (fp8_encode2(f[2], f[3], pc[1]) << 16),
                                         fp8_encode2(f[4], f[5], pc[2]) | (fp8_encode2(f[6], f[7], pc[3]) << 16)));
        }
      }
    }
  }
}

// ---- codes back to numbers ---------------------------------------------------------
// Eight codes a thread, 16 bytes stored: memory bounds it where it is large, the launch where it is small (8192 x 640 6.5 us, 2.4 TB/s).
__device__ __forceinline__ float fp8_decode(uint32_t c) {   // OCP E4M3, exactly
  uint32_t h;
  asm("{ .reg .b16 v; cvt.u16.u32 v, %1; cvt.rn.f16x2.e4m3x2 %0, v; }" : "=r"(h) : "r"(c));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}

struct DequantArgs {
  const uint8_t* codes;
  size_t code_stride;
  const float* scales;
  uint32_t rows, cols, down, across, scales_across;   // a block's height and width
  void* out;
};
template <typename T>
__global__ void __launch_bounds__(256) fp8_dequant_kernel(const __grid_constant__ DequantArgs a) {
  pdl_prologue();
  const uint32_t across = (a.cols + 7) / 8;   // eight elements a thread
  const bool wide = a.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
  const uint32_t rows_at_once = gridDim.x * 256 / across;      // a thread keeps its columns and walks down the rows, where it can
  const uint32_t t = blockIdx.x * 256 + threadIdx.x, c0 = t % across * 8;
  if (t / across >= rows_at_once) return;
  for (uint32_t row = t / across; row < a.rows; row += rows_at_once) {
    const uint8_t* src = a.codes + (size_t)row * a.code_stride + c0;
    uint2 w = make_uint2(0u, 0u);
    if (c0 + 8 <= a.cols) {
      w = *reinterpret_cast<const uint2*>(src);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c0 + k < a.cols) (k < 4 ? w.x : w.y) |= (uint32_t)src[k] << (8 * (k & 3));
    }
    const float* s = a.scales + (size_t)(row / a.down) * a.scales_across;
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      f[k] = c0 + k < a.cols ? fp8_decode(((k < 4 ? w.x : w.y) >> (8 * (k & 3))) & 0xFFu) * s[a.across == 1 ? c0 + k : c0 / kBlock] : 0.0f;
    T* out = static_cast<T*>(a.out) + (size_t)row * a.cols + c0;
    if (wide) {
      if constexpr (sizeof(T) == 2) {
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[k]) : "f"(f[2 * k + 1]), "f"(f[2 * k]));
        *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
        reinterpret_cast<float4*>(out)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(out)[1] = make_float4(f[4], f[5], f[6], f[7]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c0 + k < a.cols) {
          if constexpr (sizeof(T) == 2) out[k] = __float2bfloat16_rn(f[k]);
          else out[k] = f[k];
        }
    }
  }
}

// ---- product ------------------------------------------------------------------------
// One pass over the contraction in blocks of 128.  Roles of a thread block (12 warps):
//   warps 0-7   epilogue: per block of the contraction they read the tensor cores' sums from tensor memory (32 rows x half of the
//               columns a warp) and add them to fp32 registers with the block's scales;
//   warp 8      copies tiles of both operands to shared memory (TMA, 128-byte swizzle, out-of-range elements are zeros);
//   warps 9, 10 issue tcgen05.mma kind::f8f6f4, four of them (32 deep each) for a block of 128; each takes every other block, so that
//               one's waits pass while the other's products run;
//   warp 11     copies the blocks' scales to a ring in shared memory (asynchronous 4-byte copies, three blocks ahead).
// Operands lie in shared memory as they lie in global memory: along the contraction (K-major) or along the rows of C (MN-major,
// the weight of the input gradient and both operands of the weight gradient), which the matrix descriptor says; nothing is
// transposed.  A block's sum is scaled by one fused multiply-add a number, which is why each block needs an accumulator of its own
// in tensor memory: they take turns, so that the tensor cores work on one while another is read.
//
// What bounds it, at 8192^3 on one B200 (a pair's block of 128 is 541 cycles of products): copies and products alone take 333 us, 3.3
// PFLOP/s; with the accumulators handed to an epilogue that does nothing 383; as it is 470 (2.34 PFLOP/s) with a scale for 128 columns
// and 660 with one for each.  From a product's end to the epilogue's start pass some 420 cycles, from its release to the next product's
// start 270, between them the reading, during which products are slower: two accumulators, all that tensor memory holds, hide most of
// it.  Halves of 128 columns in four accumulators took 620 us, tiles of 256 x 192 that the epilogue reads whole before it adds 560,
// sixteen epilogue warps 500 to 510.  Power counts too: operands of zeros take 410 us, and in loops of seconds the limit of the board
// comes first (545 us at some 1.5 GHz).
//
// Two forms.  kPair, for many tiles: the two SMs of a pair work on one tile of 256 x 256 (cta_group::2), each holds half of either
// operand, the leader issues the products for both.  Without it a block has a tile of 128 x 128, and where tiles are few (serving,
// one token) a cluster of two or four blocks shares one: each takes a range of the contraction, and their sums are joined through
// distributed shared memory in the order of the ranks.
//
// Every wait gives up after two seconds.  The warp then arrives at no barrier any more, so that nothing is overwritten that another warp
// still reads and the waits of the others that depend on it give up too; an epilogue warp writes NaN for what it had not finished.  The
// kernel counts the warps (flame_fp8_product_faults), leaves its copies time to land and returns its tensor memory.
constexpr int kEpiWarps = 8;
constexpr int kProductThreads = 32 * (kEpiWarps + 4);
constexpr int kTileM = 128;                     // rows of a thread block
constexpr int kStages = 6;
constexpr int kScaleBytes = 12 * 1024;          // the ring of scales: 8 blocks of a pair's tile, 12 of a single block's
constexpr int kStagePitch = 36;                 // bytes from row to row of a warp's output staging: 32 and 4 against bank conflicts
constexpr int kStagingBytes = 32 * kStagePitch;

__device__ unsigned int g_wait_faults;

// How a product stands to the kernel before it in the stream.  kBehind: it may be placed early (a programmatic launch) and waits for it.
// kFirst, kBeside: two products of one quantiser's codes, which need nothing of each other.  The first is launched in the ordinary way: it
// starts when the quantiser is complete, and its writes visible.  The second starts when every block of the first has, so it may read the
// codes at once, and its blocks begin where the first's have ended, in place of a last round that fills a part of the SMs (4608 x 2304 x
// 9216, both gradients: 276 -> 245 us).  It reads nothing that the first writes and overwrites nothing that the first reads; it waits for
// the first before it ends, so that what waits for the second has waited for both.
enum : uint32_t { kBehind = 0, kFirst, kBeside };

struct ProductArgs {
  const float* sa;
  const float* sb;
  void* c;
  size_t c_stride;
  uint32_t M, N, K;
  uint32_t sa_stride, sb_stride;   // floats between rows of the scale arrays
  uint32_t tiles_m, tiles_n, blocks_k;
  uint32_t rows_a;                 // rows of A that a copy brings: fewer than 128 where C has fewer, a multiple of 8
  uint32_t wide;                   // rows of C start on 32 bytes
  uint32_t wide_sa, wide_sb;       // scales that lie along M or N: rows of them start on 16 bytes
  uint32_t order;                  // kBehind, kFirst or kBeside
};

struct ProductSmem {
  static constexpr int kOperand = kTileM * kBlock, kStage = 2 * kOperand;   // 128 x 128 bytes of either operand
  static constexpr int kOffScales = kStages * kStage;
  static constexpr int kOffStaging = kOffScales + kScaleBytes;
  static constexpr int kOffBars = kOffStaging + kEpiWarps * kStagingBytes;
  static constexpr int kBytes = kOffBars + 512 + 1024;                      // and room to start on 1024 bytes
};
static_assert(ProductSmem::kBytes <= 227 * 1024, "shared memory of a thread block");
static_assert(kTileM * (128 + 4) * 4 <= kStages * ProductSmem::kStage, "a tile's sums fit over the pipeline's buffers");

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ uint64_t clock_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// false: two seconds have passed, counting at most a quarter of one between two looks at the clock, which runs on while the context is
// switched out
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  uint64_t last = 0;
  uint32_t waited = 0;
  for (uint32_t n = 0;; ++n) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((n & 255u) == 255u) {
      const uint64_t now = clock_ns();
      if (last != 0) waited += now - last < 250000000ull ? (uint32_t)(now - last) : 250000000u;
      if (waited > 2000000000u) return false;
      last = now;
    }
  }
}
// kPair: the barrier may be the other block's of the pair
template <bool kPair>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  if constexpr (kPair)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: rows of 128 bytes, eight of them 1024 bytes apart from the next
// eight.  MN-major: rows of 128 elements of M or N, eight steps of the contraction 1024 bytes from the next eight, and the next 128
// elements of M or N one tile of the block behind.
template <bool kMn>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  const uint64_t lead = kMn ? (kBlock * kBlock) >> 4 : 1, stride = 1024 >> 4;
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}
template <bool kPair>
__device__ __forceinline__ void mma_fp8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (kPair)
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p; }"
                 ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
  else
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }"
                 ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// One arrival when the products issued so far are done; in a pair, at the same barrier of both blocks.
template <bool kPair>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (kPair)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// At a barrier of another block of the cluster.  Releases at the scope of this block, which orders the reads of the scales before
// their place is written again; what it tells the other block is that tensor memory has been read, which tcgen05's own fences
// order.  (A release at cluster scope took 1,300 cycles for each block of the contraction.)
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Four bytes from global to shared memory, zero where there is nothing to copy.
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4u : 0u) : "memory");
}

// Numbers of each lane, there when tmem_wait() has returned.  With a scale for 128 columns a thread takes 64 columns of one row.  With a
// scale for each column it takes the layout of 16 x 8 fragments, columns 2 (lane % 4), + 1 of rows lane / 4, + 8 in each of four
// fragments: a thread then needs the scales of a quarter of the columns, and reading them for every lane took as long as the products
// (128 bytes a cycle come from shared memory, whether or not the lanes ask for the same).
#define FLAME_R8(i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
__device__ __forceinline__ void tmem_load_row(uint32_t (&r)[64], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
               "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
               : FLAME_R8(0), FLAME_R8(8), FLAME_R8(16), FLAME_R8(24), FLAME_R8(32), FLAME_R8(40), FLAME_R8(48), FLAME_R8(56) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_load_fragments(uint32_t (&r)[16], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : FLAME_R8(0), FLAME_R8(8) : "r"(addr) : "memory");
}
#undef FLAME_R8
// The loads issued so far are done.  What uses them is volatile like this and like the loads, so that the three stay in order.
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
// acc += {lo, hi} * s, two numbers at a time
__device__ __forceinline__ void add_scaled(uint64_t& acc, uint32_t lo, uint32_t hi, uint64_t s) {
  asm volatile("{ .reg .b64 x; mov.b64 x, {%1, %2}; fma.rn.f32x2 %0, x, %3, %0; }" : "+l"(acc) : "r"(lo), "r"(hi), "l"(s));
}
// The eight pairs of four fragments: acc += (pair * scales of its columns) * scale of its row.  The products of four pairs come
// before the sums, so that none waits for the one before it.
__device__ __forceinline__ void add_scaled_fragments(uint64_t* acc, const uint32_t (&x)[16], const uint64_t (&t)[4], uint64_t s_up, uint64_t s_down) {
#pragma unroll
  for (int f = 0; f < 4; f += 2)
    asm volatile("{ .reg .b64 a, b, c, d; mov.b64 a, {%4, %5}; mov.b64 b, {%6, %7}; mov.b64 c, {%8, %9}; mov.b64 d, {%10, %11};\n\t"
                 "mul.rn.f32x2 a, a, %12; mul.rn.f32x2 b, b, %12; mul.rn.f32x2 c, c, %13; mul.rn.f32x2 d, d, %13;\n\t"
                 "fma.rn.f32x2 %0, a, %14, %0; fma.rn.f32x2 %1, b, %15, %1; fma.rn.f32x2 %2, c, %14, %2; fma.rn.f32x2 %3, d, %15, %3; }"
                 : "+l"(acc[2 * f]), "+l"(acc[2 * f + 1]), "+l"(acc[2 * f + 2]), "+l"(acc[2 * f + 3])
                 : "r"(x[4 * f]), "r"(x[4 * f + 1]), "r"(x[4 * f + 2]), "r"(x[4 * f + 3]), "r"(x[4 * f + 4]), "r"(x[4 * f + 5]), "r"(x[4 * f + 6]), "r"(x[4 * f + 7]),
                   "l"(t[f]), "l"(t[f + 1]), "l"(s_up), "l"(s_down));
}
__device__ __forceinline__ bool elect_one() {      // true in one lane of a whole warp
  uint32_t r;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const float* src, uint32_t bytes) {   // the first `bytes` of 16, then zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 peer_load4(uint32_t addr, uint32_t rank) {
  const uint32_t at = at_rank(addr, rank);
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// Tile t of C: 16 rows of tiles are walked column by column, so that the tiles in flight at a time are about as wide as high and
// their operands are read from L2.
__device__ __forceinline__ void tile_at(const ProductArgs& p, uint32_t t, uint32_t& tm, uint32_t& tn) {
  constexpr uint32_t kGroup = 16;
  const uint32_t per_group = kGroup * p.tiles_n, g = t / per_group, first = g * kGroup;
  const uint32_t high = p.tiles_m - first < kGroup ? p.tiles_m - first : kGroup;
  const uint32_t in = t - g * per_group;
  tm = first + in % high;
  tn = in / high;
}

template <typename T>
__device__ __forceinline__ uint32_t to_word(const float* v) {      // 4 bytes of C
  if constexpr (sizeof(T) == 2) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(v[1]), "f"(v[0]));
    return w;
  } else {
    return __float_as_uint(v[0]);
  }
}

template <bool kPair, bool kAmn, bool kBmn, bool kBvec, typename T>
__global__ void __launch_bounds__(kProductThreads, 1)
fp8_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ ProductArgs p) {
  using S = ProductSmem;
  constexpr int kN = kPair ? 256 : 128;                          // columns of the tile
  constexpr int kRows = kPair ? 256 : 128;                       // rows of the tile
  constexpr int kCols = kN / (kEpiWarps / 4);                                  // columns of an epilogue warp
  constexpr uint32_t kTmemCols = 512, kAccs = kTmemCols / kN;
  constexpr uint32_t kScales = (kTileM + kN) * 4, kSlots = kScaleBytes / kScales;   // scales of one block of the contraction
  // D fp32, A and B e4m3, major-ness, N / 8, M / 16
  constexpr uint32_t kIdesc = (1u << 4) | (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) | ((uint32_t)(kN / 8) << 17) | ((uint32_t)(kRows / 16) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  const uint32_t base = smem_addr(smem);
  const uint32_t bars = base + S::kOffBars;
  auto full = [&](uint32_t s) { return bars + 8 * s; };
  // One barrier says that a block's products are done, to the copies, which then may fill its stage again, as well as to the epilogue.
  // It counts the arrival of the block's scales too.
  auto done = [&](uint32_t s) { return bars + 8 * (kStages + s); };
  auto acc_empty = [&](uint32_t b) { return bars + 8 * (2 * kStages + b); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kOffBars + 8 * (2 * kStages + 4));

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t group = cluster_size(), rank = cluster_rank();  // a pair, or the blocks that share a tile's contraction
  const uint32_t splits = kPair ? 1 : group, split = kPair ? 0 : rank;
  const uint32_t worker = blockIdx.x / group, workers = gridDim.x / group;
  const uint32_t tiles = p.tiles_m * p.tiles_n;
  const uint32_t kb0 = (uint32_t)((uint64_t)p.blocks_k * split / splits), kb1 = (uint32_t)((uint64_t)p.blocks_k * (split + 1) / splits);
  const uint32_t row_off = kPair ? rank * kTileM : 0;            // of this block in the tile
  bool ok = true;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kStages; ++s) { bar_init(full(s), 1); bar_init(done(s), 2); }
    for (uint32_t b = 0; b < kAccs; ++b) bar_init(acc_empty(b), kPair ? 2 * kEpiWarps : kEpiWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kEpiWarps + 1) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (kPair) cluster_sync_all();      // the other block's barriers are ready
  tmem_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (p.order != kBeside) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // The epilogue's sums need more registers than an equal share: 384 threads start with 168 each, 64,512 together; four warps go down
  // to 72 and eight up to 216, 64,512 again.
  if (warp < kEpiWarps) {
    if constexpr (kPair) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const uint32_t quarter = warp & 3, col_off = (warp >> 2) * kCols;
    const uint32_t row = quarter * 32 + lane;
    const uint32_t release = at_rank(acc_empty(0), kPair ? 0 : rank);
    uint32_t it = 0;
    for (uint32_t t = worker; t < tiles; t += workers) {
      uint32_t tm, tn;
      tile_at(p, t, tm, tn);
      const uint32_t m0 = tm * kRows + row_off + quarter * 32;
      const uint32_t n0 = tn * kN + col_off;
      const bool live = m0 < p.M && n0 < p.N;
      uint64_t acc2[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) acc2[i] = 0ull;
      for (uint32_t kb = ok ? kb0 : kb1; kb < kb1; ++kb, ++it) {
        const uint32_t b = it % kAccs;
        ok = ok && bar_wait(done(it % kStages), (it / kStages) & 1);      // after a wait that ran out none is waited for: the loop runs to its end
        __syncwarp();
        tmem_fence_after();
        if (live) {
          const uint32_t src = tmem + b * kN + col_off + (quarter << 21);   // lane 32 * quarter in the upper 16 bits
          const float* sc = reinterpret_cast<const float*>(smem + S::kOffScales + it % kSlots * kScales);
          auto free_accumulator = [&]() {       // all is in registers
            tmem_fence_before();
            __syncwarp();
            if (lane == 0 && ok) bar_arrive_cluster(release + 8 * b);
          };
          if constexpr (kBvec) {
            // piece k: 32 columns of the thread's four fragments in 16 of the warp's rows; one on its way while another is added
            uint32_t v[2][16];
            auto piece = [&](int k) { return src + k / 2 * 32 + ((uint32_t)(k % 2) << 20); };
            tmem_load_fragments(v[0], piece(0));
            uint64_t sa[4], sb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { const uint32_t w = __float_as_uint(sc[quarter * 32 + i * 8 + lane / 4]); sa[i] = pack2(w, w); }
#pragma unroll
            for (int k = 0; k < kCols / 16; ++k) {
              tmem_wait();
              if (k + 1 < kCols / 16) tmem_load_fragments(v[k % 2 ^ 1], piece(k + 1));
              else free_accumulator();
              if (k % 2 == 0) {
#pragma unroll
                for (int f = 0; f < 4; ++f) sb[f] = *reinterpret_cast<const uint64_t*>(sc + kTileM + col_off + k / 2 * 32 + f * 8 + lane % 4 * 2);
              }
              add_scaled_fragments(acc2 + 8 * k, v[k % 2], sb, sa[k % 2 * 2], sa[k % 2 * 2 + 1]);
            }
          } else {
            // 64 columns at a time and none on its way meanwhile: what counts is how soon the accumulator is free again, and pieces of 16
            // that overlap with the multiply-adds free it later (8192^3: 490 us against 470).  With a scale for each column the multiply-adds
            // take twice as long, and overlapping them wins (4096^3, rows: 129 us against 146).
            uint32_t x[64];
            tmem_load_row(x, src);
            const uint32_t w = __float_as_uint(sc[row] * sc[kTileM + col_off / kBlock]);
            const uint64_t s = pack2(w, w);
#pragma unroll
            for (int k = 0; k < kCols / 64; ++k) {
              tmem_wait();
              if (k + 1 == kCols / 64) free_accumulator();
#pragma unroll
              for (int i = 0; i < 32; ++i) add_scaled(acc2[32 * k + i], x[2 * i], x[2 * i + 1], s);
              if (k + 1 < kCols / 64) tmem_load_row(x, src + (k + 1) * 64);
            }
          }
        } else if (lane == 0 && ok) {
          bar_arrive_cluster(release + 8 * b);
        }
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) {
#pragma unroll
        for (int i = 0; i < kCols / 2; ++i) acc2[i] = pack2(0x7FC00000u, 0x7FC00000u);
      }
      if (kPair || splits == 1) {
        if (!live) continue;
        constexpr int kPer = 32 / sizeof(T);       // columns in 32 bytes
        const uint32_t rows = p.M - m0 < 32 ? p.M - m0 : 32;
        T* out = static_cast<T*>(p.c) + (size_t)m0 * p.c_stride + n0;
        uint8_t* st = smem + S::kOffStaging + warp * kStagingBytes;
        const uint8_t* my_row = st + lane * kStagePitch;
#pragma unroll
        for (int c = 0; c < kCols; c += kPer) {
          if (n0 + c >= p.N) break;
          const bool wide = p.wide && n0 + c + kPer <= p.N;
          uint32_t w[8];
          if constexpr (kBvec) {
            // fragments: two neighbouring columns of four rows
#pragma unroll
            for (int f = 0; f < kPer / 8; ++f)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int nb = c / 8 + f;          // fragment column of the warp, rows i * 8 + lane / 4
                const float2 u = unpack2(acc2[(nb / 4 * 2 + i / 2) * 8 + nb % 4 * 2 + i % 2]);
                uint8_t* at = st + (i * 8 + lane / 4) * kStagePitch + f * 8 * sizeof(T) + lane % 4 * 2 * sizeof(T);
                const float pair[2] = {u.x, u.y};
                *reinterpret_cast<uint32_t*>(at) = to_word<T>(pair);
                if (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(at + 4) = __float_as_uint(u.y);
              }
            __syncwarp();
            if (wide) {
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint32_t*>(my_row + 4 * i);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 u = unpack2(acc2[sizeof(T) == 2 ? c / 2 + i : (c + i) / 2]);
              const float pair[2] = {sizeof(T) == 2 || i % 2 == 0 ? u.x : u.y, u.y};
              w[i] = to_word<T>(pair);
            }
            if (!wide) {
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(st + lane * kStagePitch + 4 * i) = w[i];
              __syncwarp();
            }
          }
          if (wide) {
            // a whole sector of a row from each lane
            if (lane < rows)
              asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + (size_t)lane * p.c_stride + c), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                           "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
          } else {
            // rows that start anywhere: neighbouring lanes write neighbouring columns
            const uint32_t cols = p.N - (n0 + c) < (uint32_t)kPer ? p.N - (n0 + c) : kPer, j = lane % kPer;
            if (j < cols)
              for (uint32_t r = lane / kPer; r < rows; r += 32 / kPer) out[(size_t)r * p.c_stride + c + j] = reinterpret_cast<const T*>(st + r * kStagePitch)[j];
          }
          __syncwarp();
        }
      } else if (live) {
        // this block's share of the tile, over the pipeline's buffers: every copy has landed and every product has been read
        float* mine = reinterpret_cast<float*>(smem) + (size_t)(quarter * 32) * (kN + 4) + col_off;
        if constexpr (kBvec) {
#pragma unroll
          for (int k = 0; k < kCols / 16; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float2*>(mine + (k % 2 * 16 + i % 2 * 8 + lane / 4) * (kN + 4) + k / 2 * 32 + i / 2 * 8 + lane % 4 * 2) = unpack2(acc2[8 * k + i]);
        } else {
#pragma unroll
          for (int i = 0; i < kCols / 2; i += 2) {
            const float2 u = unpack2(acc2[i]), v = unpack2(acc2[i + 1]);
            *reinterpret_cast<float4*>(mine + lane * (kN + 4) + 2 * i) = make_float4(u.x, u.y, v.x, v.y);
          }
        }
      }
    }
  } else {
    if constexpr (kPair) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kEpiWarps) {
      if (lane == 0) {
        uint32_t it = 0;
        for (uint32_t t = worker; t < tiles; t += workers) {
          uint32_t tm, tn;
          tile_at(p, t, tm, tn);
          const int32_t m = (int32_t)(tm * kRows + row_off), n = (int32_t)(tn * kN + (kPair ? rank * kBlock : 0));
          for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
            const uint32_t s = it % kStages;
            if (!(ok = ok && bar_wait(done(s), ((it / kStages) & 1) ^ 1))) continue;
            // the leader's barrier counts the bytes of both blocks
            if (!kPair || rank == 0) bar_expect(full(s), kPair ? 2 * S::kStage : S::kOperand + (kAmn ? S::kOperand : p.rows_a * kBlock));
            const uint32_t bar = kPair ? at_rank(full(s), 0) : full(s);
            const uint32_t sa = base + s * S::kStage, sb = sa + S::kOperand;
            const int32_t k = (int32_t)(kb * kBlock);
            tma_load<kPair>(sa, &map_a, kAmn ? m : k, kAmn ? k : m, bar);
            tma_load<kPair>(sb, &map_b, kBmn ? n : k, kBmn ? k : n, bar);
          }
        }
      }
    } else if (warp <= kEpiWarps + 2) {
      if (!kPair || rank == 0) {
        // The whole warp walks the loop and one lane issues: descriptors then come from the warp's uniform registers.  (In a branch of one
        // lane each had to be moved there from a lane's, and a block's four products took 480 cycles to issue.)
        const uint32_t mine = tiles > worker ? (tiles - worker + workers - 1) / workers * (kb1 - kb0) : 0;   // of all the block's tiles
        const uint32_t issuer = __shfl_sync(0xFFFFFFFFu, warp, 0) - (kEpiWarps + 1);
        for (uint32_t it = issuer; it < mine; it += 2) {
          const uint32_t s = it % kStages, b = it % kAccs;
          ok = ok && bar_wait(full(s), (it / kStages) & 1) && bar_wait(acc_empty(b), ((it / kAccs) & 1) ^ 1);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          tmem_fence_after();
          // 32 deep a step: 32 bytes along a K-major row, 32 rows of 128 bytes of an MN-major tile
          const uint64_t da = smem_desc<kAmn>(base + s * S::kStage), db = smem_desc<kBmn>(base + s * S::kStage + S::kOperand);
          const uint32_t acc = tmem + b * kN, at_done = done(s);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kBlock / 32; ++j)
              mma_fp8<kPair>(acc, da + (uint64_t)(j * (kAmn ? 32 * kBlock : 32) >> 4), db + (uint64_t)(j * (kBmn ? 32 * kBlock : 32) >> 4), kIdesc, j > 0);
            mma_commit<kPair>(at_done);
          }
          __syncwarp();
        }
      }
    } else {
      // Copies run kAhead blocks ahead.  When block i - kAccs has its products, every warp of the epilogue has given the accumulator of
      // block i - 2 kAccs back, which it does after its last use of the scales of the block before that: their place in the ring is
      // free for block i + kSlots - 2 kAccs - 1's.
      constexpr uint32_t kAhead = kSlots - 2 * kAccs - 1;
      static_assert(kAhead == 3, "8 places for two accumulators, 12 for four");
      uint32_t t_copy = worker, kb_copy = kb1, slot_at = base + S::kOffScales, a_left = 0, b_left = 0;
      const float *pa = p.sa, *pb = p.sb;
      // from one row (column) of the tile to the 32nd after it, and from one block of the contraction to the next
      const size_t a32 = kAmn ? 32 : 32 * (size_t)p.sa_stride, b32 = kBmn ? 32 : 32 * (size_t)p.sb_stride;
      const bool wide_a = kAmn && p.wide_sa, wide_b = kBvec && kBmn && p.wide_sb;
      auto copy_next = [&]() {
        if (kb_copy == kb1 && t_copy < tiles) {      // a new tile: this lane's first row and column of scales
          uint32_t tm, tn;
          tile_at(p, t_copy, tm, tn);
          t_copy += workers;
          kb_copy = kb0;
          // the lane's first row (and column) of scales: every 32nd, or where they are neighbours in memory four together
          const uint32_t la = wide_a ? 4 * lane : lane, lb = wide_b ? 4 * lane : lane;
          const uint32_t m = tm * kRows + row_off + la, n = kBvec ? tn * kN + lb : tn * (kN / kBlock) + lb;
          const uint32_t n_end = kBvec ? p.N : (p.N + kBlock - 1) / kBlock;
          a_left = m < p.M ? p.M - m : 0;
          b_left = n < n_end ? n_end - n : 0;
          pa = p.sa + (a_left == 0 ? 0 : kAmn ? (size_t)kb0 * p.sa_stride + m : (size_t)m * p.sa_stride + kb0);
          pb = p.sb + (b_left == 0 ? 0 : kBmn ? (size_t)kb0 * p.sb_stride + n : (size_t)n * p.sb_stride + kb0);
        }
        if (kb_copy < kb1) {
          if (wide_a) {
            copy16(slot_at + lane * 16, pa, a_left < 4 ? a_left * 4 : 16);
          } else {
#pragma unroll
            for (uint32_t i = 0; i < kTileM / 32; ++i) copy4(slot_at + (i * 32 + lane) * 4, i * 32 < a_left ? pa + i * a32 : p.sa, i * 32 < a_left);
          }
          if constexpr (kBvec) {
            if (wide_b) {
#pragma unroll
              for (uint32_t i = 0; i < kN / 128; ++i) {
                const uint32_t left = b_left > i * 128 ? b_left - i * 128 : 0;
                copy16(slot_at + (kTileM + i * 128) * 4 + lane * 16, left ? pb + i * 128 : p.sb, left < 4 ? left * 4 : 16);
              }
            } else {
#pragma unroll
              for (uint32_t i = 0; i < kN / 32; ++i) copy4(slot_at + (kTileM + i * 32 + lane) * 4, i * 32 < b_left ? pb + i * b32 : p.sb, i * 32 < b_left);
            }
          } else if (lane < kN / kBlock) {
            copy4(slot_at + (kTileM + lane) * 4, b_left ? pb : p.sb, b_left != 0);
          }
          if (a_left) pa += kAmn ? p.sa_stride : 1;
          if (b_left) pb += kBmn ? p.sb_stride : 1;
          ++kb_copy;
        }
        slot_at = slot_at + kScales == base + S::kOffScales + kSlots * kScales ? base + S::kOffScales : slot_at + kScales;
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      for (uint32_t i = 0; i < kAhead; ++i) copy_next();
      uint32_t it = 0;
      for (uint32_t t = worker; t < tiles; t += workers)
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
          if (it >= kAccs) ok = ok && bar_wait(done((it - kAccs) % kStages), ((it - kAccs) / kStages) & 1);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) continue;
          copy_next();
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");   // block `it` has landed
          __syncwarp();
          if (lane == 0) bar_arrive(done(it % kStages));
        }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  }

  if (__any_sync(0xFFFFFFFFu, !ok)) {      // a wait ran out: the copies and products in flight get a millisecond to end
    const uint64_t since = clock_ns();
    while (clock_ns() - since < 1000000ull) {}
    if (lane == 0) atomicAdd(&g_wait_faults, 1u);
    if (!kPair && splits > 1 && warp < kEpiWarps) {      // the share that lies over the pipeline's buffers, now that no copy lands there
      float* mine = reinterpret_cast<float*>(smem) + (size_t)((warp & 3) * 32 + lane) * (kN + 4) + (warp >> 2) * kCols;
      for (int i = 0; i < kCols; ++i) mine[i] = __uint_as_float(0x7FC00000u);
    }
  }
  __syncwarp();
  if (!kPair && splits > 1) {      // one tile for each cluster
    cluster_sync_all();
    if (warp < kEpiWarps && worker < tiles) {
      uint32_t tm, tn;
      tile_at(p, worker, tm, tn);
      constexpr uint32_t kEpiThreads = 32 * kEpiWarps;
      const uint32_t rows = p.M - tm * kTileM < (uint32_t)kTileM ? p.M - tm * kTileM : kTileM;
      for (uint32_t i = rank * kEpiThreads + threadIdx.x; i < rows * (kN / 4); i += splits * kEpiThreads) {
        const uint32_t r = i / (kN / 4), c = i % (kN / 4) * 4, n = tn * kN + c;
        if (n >= p.N) continue;
        const uint32_t at = base + (r * (kN + 4) + c) * 4;
        float4 sum = peer_load4(at, 0);
        for (uint32_t k = 1; k < splits; ++k) {
          const float4 v = peer_load4(at, k);
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        T* out = static_cast<T*>(p.c) + (size_t)(tm * kTileM + r) * p.c_stride + n;
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) {
            if constexpr (sizeof(T) == 2) out[j] = __float2bfloat16_rn(f[j]);
            else out[j] = f[j];
          }
      }
    }
    __syncwarp();
  }
  tmem_fence_before();
  __syncthreads();
  if (kPair || splits > 1) cluster_sync_all();   // nobody's shared or tensor memory goes away while another block of the cluster uses it
  tmem_fence_after();
  if (warp == kEpiWarps + 1) {
    if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  if (p.order == kBeside) asm volatile("griddepcontrol.wait;" ::: "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}
// rows x cols bytes, `stride` bytes from row to row, copied as 128 columns x `high` rows
bool byte_matrix(CUtensorMap* map, const uint8_t* p, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t high) {
  const EncodeTiled f = encode_tiled();
  if (!f) return false;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {stride};
  const cuuint32_t box[2] = {kBlock, high}, one[2] = {1, 1};
  return f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operands {
  const uint8_t* a;
  const uint8_t* b;
  size_t a_stride, b_stride;
};

template <bool kPair, bool kAmn, bool kBmn, bool kBvec, typename T>
cudaError_t launch_tiles(const Operands& o, const ProductArgs& p, uint32_t group, uint32_t blocks, cudaStream_t stream) {
  CUtensorMap map_a, map_b;
  const bool ok = byte_matrix(&map_a, o.a, kAmn ? p.K : p.M, kAmn ? p.M : p.K, o.a_stride, kAmn ? kBlock : p.rows_a) &&
                  byte_matrix(&map_b, o.b, kBmn ? p.K : p.N, kBmn ? p.N : p.K, o.b_stride, kBlock);
  if (!ok) return cudaErrorNotSupported;
  auto kern = fp8_product_kernel<kPair, kAmn, kBmn, kBvec, T>;
  static std::atomic<uint64_t> allowed{0};     // a bit for each device on which the kernel may use this much shared memory
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    if (const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ProductSmem::kBytes)) return e;
    if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kProductThreads);
  cfg.dynamicSmemBytes = ProductSmem::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (group > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = group;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.order != kFirst && pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, map_a, map_b, p);
}

template <bool kAmn, bool kBmn, bool kBvec, typename T>
cudaError_t launch_product_t(const Operands& o, ProductArgs p, cudaStream_t stream) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  p.blocks_k = (p.K + kBlock - 1) / kBlock;
  p.wide = (reinterpret_cast<uintptr_t>(p.c) & 31u) == 0 && (p.c_stride * sizeof(T)) % 32 == 0;
  // Rows of C that do not exist: what their rows of A hold in shared memory reaches no other row of C and is not stored, so a copy
  // leaves them out (one token against 8192 x 8192: 18.3 -> 14.4 us; out-of-range rows of a copy are written as zeros and take time).
  p.rows_a = p.M < (uint32_t)kTileM ? (p.M + 7) / 8 * 8 : kTileM;
  p.wide_sa = kAmn && (reinterpret_cast<uintptr_t>(p.sa) & 15u) == 0 && p.sa_stride % 4 == 0;
  p.wide_sb = kBmn && kBvec && (reinterpret_cast<uintptr_t>(p.sb) & 15u) == 0 && p.sb_stride % 4 == 0;
  // Which form: a round of pairs (256 x 256 tiles, one for two SMs) takes 1.0 where a round of single blocks (128 x 128) takes 0.70,
  // measured with one round of each: 2048 x 2048 and 1536 x 1536 took 18.8 and 13.2 us at K = 4096, 9.0 and 6.0 us at K = 1024.  The 16
  // tiles of one token against 2048 x 2048 took 5.2 us with four blocks to a tile, 6.0 with two, 7.5 with one and 9.3 with eight:
  // clusters of eight wait for a place.
  const uint64_t pairs = (uint64_t)sms / 2, rounds_of_pairs = ((uint64_t)((p.M + 255) / 256) * ((p.N + 255) / 256) + pairs - 1) / pairs;
  p.tiles_m = (p.M + 127) / 128;
  p.tiles_n = (p.N + 127) / 128;
  const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n, rounds = (tiles + sms - 1) / sms;
  uint32_t splits = 1;
  while (splits < 4 && tiles * splits * 2 <= (uint64_t)sms && splits * 2 <= p.blocks_k) splits *= 2;
  if (splits == 1 && rounds_of_pairs * 100 <= rounds * 70) {
    p.tiles_m = (p.M + 255) / 256;
    p.tiles_n = (p.N + 255) / 256;
    p.rows_a = kTileM;
    return launch_tiles<true, kAmn, kBmn, kBvec, T>(o, p, 2, (uint32_t)(2 * pairs), stream);
  }
  const uint32_t blocks = splits > 1 ? (uint32_t)tiles * splits : (uint32_t)(tiles < (uint64_t)sms ? tiles : (uint64_t)sms);
  return launch_tiles<false, kAmn, kBmn, kBvec, T>(o, p, splits, blocks, stream);
}

template <bool kAmn, bool kBmn, bool kBvec>
cudaError_t launch_product(const Operands& o, const ProductArgs& p, bool f32, cudaStream_t s) {
  return f32 ? launch_product_t<kAmn, kBmn, kBvec, float>(o, p, s) : launch_product_t<kAmn, kBmn, kBvec, __nv_bfloat16>(o, p, s);
}

bool al(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
int refuse(const char* who, const char* what) {
  set_last_error(std::string(who) + ": " + what);
  return (int)cudaErrorInvalidValue;
}
constexpr uint64_t kMostSize = 0x7FFFFFFFull / 2;
size_t up16(size_t n) { return n == 0 ? 16 : (n + 15) / 16 * 16; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
uint64_t blocks_of(uint64_t n) { return (n + kBlock - 1) / kBlock; }
// codes and, on the next 256 bytes, scales
size_t codes_bytes(size_t rows, size_t cols, uint32_t mode) {
  const size_t scales = mode == kQuantColumns ? blocks_of(rows) * cols : mode == kQuantTiles ? blocks_of(rows) * blocks_of(cols) : rows * blocks_of(cols);
  return up256(rows * up16(cols)) + up256(scales * sizeof(float));
}

// What is wrong with a BF16 matrix as a source of codes; NULL: nothing.
const char* quant_source(const void* x, size_t rows, size_t cols, size_t stride) {
  if (rows > kMostSize || cols > kMostSize || blocks_of(rows) * blocks_of(cols) > 0x3FFFFFFFull) return "matrix too large";
  if (stride < cols) return "a stride is smaller than the row";
  if (rows == 0 || cols == 0) return nullptr;
  if (!x) return "null tensor";
  return al(x, 2) ? nullptr : "misaligned tensor";
}
QuantJob quant_job(const void* x, size_t rows, size_t cols, size_t x_stride, uint32_t mode, void* row_codes, void* row_scales, void* col_codes, void* col_scales,
                   size_t code_stride) {
  QuantJob a;
  a.x = static_cast<const __nv_bfloat16*>(x); a.x_stride = x_stride; a.rows = (uint32_t)rows; a.cols = (uint32_t)cols;
  a.row_codes = static_cast<uint8_t*>(row_codes); a.row_scales = static_cast<float*>(row_scales);
  a.col_codes = static_cast<uint8_t*>(col_codes); a.col_scales = static_cast<float*>(col_scales);
  a.code_stride = code_stride; a.tiles_across = (uint32_t)blocks_of(cols);
  a.tiles = (uint32_t)(blocks_of(rows) * blocks_of(cols));
  a.mode = mode | (al(x, 16) && x_stride % 8 == 0 && cols % 8 == 0 ? kQuantWide : 0u);
  return a;
}
cudaError_t launch_quant(const QuantJobs& jobs, cudaStream_t stream) {
  const uint64_t tiles = (uint64_t)jobs.job[0].tiles + jobs.job[1].tiles + jobs.job[2].tiles;
  if (tiles > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
  return tiles == 0 ? cudaSuccess : launch_after(fp8_quant_kernel, (unsigned)tiles, kQuantThreads, 0, stream, jobs);
}
// Where a matrix's codes and scales lie in a workspace; moves `at` on.
struct Place { uint8_t *codes, *scales; };
Place take(uint8_t*& at, size_t rows, size_t cols, uint32_t mode) {
  const Place p = {at, at + up256(rows * up16(cols))};
  at += codes_bytes(rows, cols, mode);
  return p;
}

enum class Product { kNtTiles, kNtRows, kNnTiles, kTnColumns };
cudaError_t product(Product kind, const void* a, size_t a_stride, const void* sa, const void* b, size_t b_stride, const void* sb, void* c, size_t c_stride, bool f32,
                    size_t M, size_t N, size_t K, cudaStream_t s, uint32_t order = kBehind) {
  if (blocks_of(M) * blocks_of(N) > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;      // a result of over 2^45 numbers
  if (K == 0) {   // an empty sum
    const size_t size = f32 ? 4 : 2;
    return cudaMemset2DAsync(c, c_stride * size, 0, N * size, M, s);
  }
  const Operands o = {static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), a_stride, b_stride};
  ProductArgs p = {};
  p.sa = static_cast<const float*>(sa); p.sb = static_cast<const float*>(sb);
  p.c = c; p.c_stride = c_stride; p.order = order;
  p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K;
  p.sa_stride = kind == Product::kTnColumns ? (uint32_t)M : (uint32_t)blocks_of(K);
  p.sb_stride = kind == Product::kTnColumns ? (uint32_t)N : (uint32_t)blocks_of(kind == Product::kNnTiles ? N : K);
  if (kind == Product::kNtTiles) return launch_product<false, false, false>(o, p, f32, s);
  if (kind == Product::kNtRows) return launch_product<false, false, true>(o, p, f32, s);
  if (kind == Product::kNnTiles) return launch_product<false, true, false>(o, p, f32, s);
  return launch_product<true, true, true>(o, p, f32, s);
}

}  // namespace
}  // namespace flame_b200

using namespace flame_b200;

extern "C" {

int flame_fp8_quant_2d(const void* x, size_t rows, size_t cols, size_t x_stride, void* codes, void* scales, int blocks,
                       void* column_codes, void* column_scales, size_t code_stride, void* stream) {
  const char* who = "flame_fp8_quant_2d";
  const bool tile = blocks == FLAME_FP8_BLOCKS_TILES, row = blocks == FLAME_FP8_BLOCKS_ROWS, col = column_codes != nullptr;
  if (!tile && !row && blocks != 0) return refuse(who, "blocks must be 0, FLAME_FP8_BLOCKS_ROWS or FLAME_FP8_BLOCKS_TILES");
  if (tile && col) return refuse(who, "tiles and columns are not made in one call");
  if (const char* what = quant_source(x, rows, cols, x_stride)) return refuse(who, what);
  if (code_stride < cols || code_stride % 16 != 0) return refuse(who, "the code stride is smaller than the row, or no multiple of 16");
  if (rows == 0 || cols == 0) return 0;
  if (!tile && !row && !col) return refuse(who, "nothing to make");
  if (((tile || row) && (!codes || !scales)) || (col && !column_scales)) return refuse(who, "null tensor");
  if (!al(codes, 16) || !al(column_codes, 16) || !al(scales, 4) || !al(column_scales, 4)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  const QuantJob a = quant_job(x, rows, cols, x_stride, (tile ? kQuantTiles : 0u) | (row ? kQuantRows : 0u) | (col ? kQuantColumns : 0u), codes, scales,
                               column_codes, column_scales, code_stride);
  QuantJobs jobs = {};
  jobs.job[0] = a;
  return cuda_result(who, launch_quant(jobs, (cudaStream_t)stream));
}

int flame_fp8_dequant_2d(const void* codes, size_t code_stride, const void* scales, int blocks, void* out, int out_dtype, size_t rows,
                         size_t cols, void* stream) {
  const char* who = "flame_fp8_dequant_2d";
  if (blocks != FLAME_FP8_BLOCKS_ROWS && blocks != FLAME_FP8_BLOCKS_COLUMNS && blocks != FLAME_FP8_BLOCKS_TILES) return refuse(who, "unknown blocks");
  if (out_dtype != FLAME_OFFLOAD_DTYPE_BF16 && out_dtype != FLAME_OFFLOAD_DTYPE_F32) return refuse(who, "the output is BF16 or F32");
  if (rows > kMostSize || cols > kMostSize) return refuse(who, "matrix too large");
  if (code_stride < cols || code_stride % 16 != 0) return refuse(who, "the code stride is smaller than the row or no multiple of 16");
  if (rows == 0 || cols == 0) return 0;
  if (!codes || !scales || !out) return refuse(who, "null tensor");
  if (!al(codes, 16) || !al(scales, 4) || !al(out, out_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  DequantArgs a;
  a.codes = static_cast<const uint8_t*>(codes); a.code_stride = code_stride; a.scales = static_cast<const float*>(scales);
  a.rows = (uint32_t)rows; a.cols = (uint32_t)cols; a.out = out;
  a.down = blocks == FLAME_FP8_BLOCKS_ROWS ? 1 : kBlock;
  a.across = blocks == FLAME_FP8_BLOCKS_COLUMNS ? 1 : kBlock;
  a.scales_across = blocks == FLAME_FP8_BLOCKS_COLUMNS ? (uint32_t)cols : (uint32_t)((cols + 127) / 128);
  // at least one row of threads, so that every column has one
  const uint64_t across = (cols + 7) / 8, wanted = ((uint64_t)rows * across + 255) / 256, least = (across + 255) / 256;
  const unsigned grid = (unsigned)(wanted < 148 * 32 ? wanted : least > 148 * 32 ? least : 148 * 32);
  return cuda_result(who, out_dtype == FLAME_OFFLOAD_DTYPE_F32 ? launch_after(fp8_dequant_kernel<float>, grid, 256, 0, (cudaStream_t)stream, a)
                                                               : launch_after(fp8_dequant_kernel<__nv_bfloat16>, grid, 256, 0, (cudaStream_t)stream, a));
}

int flame_fp8_product(const void* a_codes, size_t a_stride, const void* a_scales, int a_blocks, const void* b_codes, size_t b_stride,
                      const void* b_scales, int b_blocks, int b_transposed, void* c, size_t c_stride, int c_dtype, size_t M, size_t N, size_t K, void* stream) {
  const char* who = "flame_fp8_product";
  Product kind;
  if (a_blocks == FLAME_FP8_BLOCKS_ROWS && b_blocks == FLAME_FP8_BLOCKS_TILES) kind = b_transposed ? Product::kNtTiles : Product::kNnTiles;
  else if (a_blocks == FLAME_FP8_BLOCKS_ROWS && b_blocks == FLAME_FP8_BLOCKS_ROWS && b_transposed) kind = Product::kNtRows;
  else if (a_blocks == FLAME_FP8_BLOCKS_COLUMNS && b_blocks == FLAME_FP8_BLOCKS_COLUMNS && !b_transposed) kind = Product::kTnColumns;
  else return refuse(who, "the blocks of both operands must run along the contraction: rows x rows^T, rows x tiles^T, rows x tiles or columns^T x columns");
  if (c_dtype != FLAME_OFFLOAD_DTYPE_BF16 && c_dtype != FLAME_OFFLOAD_DTYPE_F32) return refuse(who, "the output is BF16 or F32");
  if (M > kMostSize || N > kMostSize || K > kMostSize) return refuse(who, "matrix too large");
  const size_t a_row = kind == Product::kTnColumns ? M : K, b_row = b_transposed ? K : N;
  if (a_stride < a_row || b_stride < b_row || a_stride % 16 != 0 || b_stride % 16 != 0 || c_stride < N) return refuse(who, "a stride is smaller than its row, or a code stride no multiple of 16");
  if (M == 0 || N == 0) return 0;
  if (!c || !al(c, c_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2)) return refuse(who, "null or misaligned output");
  if (K != 0 && (!a_codes || !b_codes || !a_scales || !b_scales)) return refuse(who, "null tensor");
  if (!al(a_codes, 16) || !al(b_codes, 16) || !al(a_scales, 4) || !al(b_scales, 4)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  return cuda_result(who, product(kind, a_codes, a_stride, a_scales, b_codes, b_stride, b_scales, c, c_stride, c_dtype == FLAME_OFFLOAD_DTYPE_F32, M, N, K, (cudaStream_t)stream));
}

size_t flame_fp8_linear_workspace_bytes(size_t M, size_t N, size_t K, int flags) {
  if (M > kMostSize || N > kMostSize || K > kMostSize) return 0;
  const size_t w = (flags & FLAME_FP8_LINEAR_BF16_WEIGHT) ? codes_bytes(N, K, kQuantTiles) : 0;
  if (!(flags & FLAME_FP8_LINEAR_BACKWARD)) return codes_bytes(M, K, kQuantRows) + w;
  return codes_bytes(M, N, kQuantRows) + codes_bytes(M, N, kQuantColumns) + codes_bytes(M, K, kQuantColumns) + w;
}

int flame_fp8_linear(const void* x, size_t x_stride, const void* x_codes, size_t x_code_stride, const void* x_scales, const void* w,
                     size_t w_stride, const void* w_codes, size_t w_code_stride, const void* w_scales, int w_blocks, void* y, size_t M,
                     size_t N, size_t K, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "flame_fp8_linear";
  if (!w && w_blocks != FLAME_FP8_BLOCKS_TILES && w_blocks != FLAME_FP8_BLOCKS_ROWS) return refuse(who, "the blocks of a weight are tiles or rows");
  if (const char* what = x_codes ? nullptr : quant_source(x, M, K, x_stride)) return refuse(who, what);
  if (const char* what = w ? quant_source(w, N, K, w_stride) : nullptr) return refuse(who, what);
  if (M > kMostSize || N > kMostSize || K > kMostSize) return refuse(who, "matrix too large");
  if ((!w && (w_code_stride < K || w_code_stride % 16 != 0)) || (x_codes && (x_code_stride < K || x_code_stride % 16 != 0)))
    return refuse(who, "a code stride is smaller than the row, or no multiple of 16");
  if (N == 0 || M == 0) return 0;
  if (!y || (x_codes && !x_scales) || (K > 0 && !w && (!w_codes || !w_scales))) return refuse(who, "null tensor");
  if (!al(y, 2) || !al(w_codes, 16) || !al(w_scales, 4) || !al(x_codes, 16) || !al(x_scales, 4)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  if (K > 0 && (!x_codes || w) && (!workspace || !al(workspace, 256) || workspace_bytes < flame_fp8_linear_workspace_bytes(M, N, K, w ? FLAME_FP8_LINEAR_BF16_WEIGHT : 0)))
    return refuse(who, "workspace too small, or not on 256 bytes");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  cudaStream_t s = (cudaStream_t)stream;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  QuantJobs jobs = {};
  if (!x_codes && K > 0) {
    const Place q = take(at, M, K, kQuantRows);
    x_code_stride = up16(K);
    x_codes = q.codes;
    x_scales = q.scales;
    jobs.job[0] = quant_job(x, M, K, x_stride, kQuantRows, q.codes, q.scales, nullptr, nullptr, x_code_stride);
  }
  if (w && K > 0) {
    const Place q = take(at, N, K, kQuantTiles);
    w_code_stride = up16(K);
    w_codes = q.codes;
    w_scales = q.scales;
    jobs.job[1] = quant_job(w, N, K, w_stride, kQuantTiles, q.codes, q.scales, nullptr, nullptr, w_code_stride);
  }
  if (const cudaError_t e = launch_quant(jobs, s)) return cuda_result(who, e);
  return cuda_result(who, product(w || w_blocks == FLAME_FP8_BLOCKS_TILES ? Product::kNtTiles : Product::kNtRows, x_codes, x_code_stride, x_scales, w_codes, w_code_stride,
                                  w_scales, y, N, false, M, N, K, s));
}

int flame_fp8_linear_backward(const void* dy, size_t dy_stride, const void* x, size_t x_stride, const void* w, size_t w_stride, const void* w_codes,
                              size_t w_code_stride, const void* w_scales, void* dx, void* dw, size_t M, size_t N, size_t K, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* who = "flame_fp8_linear_backward";
  if (const char* what = quant_source(dy, M, N, dy_stride)) return refuse(who, what);
  if (const char* what = dw ? quant_source(x, M, K, x_stride) : nullptr) return refuse(who, what);
  if (const char* what = dx && w ? quant_source(w, N, K, w_stride) : nullptr) return refuse(who, what);
  if (K > kMostSize) return refuse(who, "matrix too large");
  if (dx && !w && (w_code_stride < K || w_code_stride % 16 != 0)) return refuse(who, "a code stride is smaller than the row, or no multiple of 16");
  if ((!dx && !dw) || K == 0) return 0;
  const bool any = M > 0 && N > 0;
  if (any && dx && !w && (!w_codes || !w_scales)) return refuse(who, "null tensor");
  if (!al(dx, 2) || !al(dw, 2) || !al(w_codes, 16) || !al(w_scales, 4)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  if (any && (!workspace || !al(workspace, 256) ||
              workspace_bytes < flame_fp8_linear_workspace_bytes(M, N, K, FLAME_FP8_LINEAR_BACKWARD | (w ? FLAME_FP8_LINEAR_BF16_WEIGHT : 0))))
    return refuse(who, "workspace too small, or not on 256 bytes");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return cuda_result(who, cudaErrorLaunchFailure);
  cudaStream_t s = (cudaStream_t)stream;
  const size_t ldn = up16(N), ldk = up16(K);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  Place rows = {}, cols = {}, xcols = {};
  if (any) {
    rows = take(at, M, N, kQuantRows);
    cols = take(at, M, N, kQuantColumns);
    xcols = take(at, M, K, kQuantColumns);
    QuantJobs jobs = {};
    jobs.job[0] = quant_job(dy, M, N, dy_stride, (dx ? kQuantRows : 0u) | (dw ? kQuantColumns : 0u), rows.codes, rows.scales, cols.codes, cols.scales, ldn);
    if (dw) jobs.job[1] = quant_job(x, M, K, x_stride, kQuantColumns, nullptr, nullptr, xcols.codes, xcols.scales, ldk);
    if (dx && w) {
      const Place q = take(at, N, K, kQuantTiles);
      jobs.job[2] = quant_job(w, N, K, w_stride, kQuantTiles, q.codes, q.scales, nullptr, nullptr, ldk);
      w_codes = q.codes;
      w_code_stride = ldk;
      w_scales = q.scales;
    }
    if (const cudaError_t e = launch_quant(jobs, s)) return cuda_result(who, e);
  }
  // the two side by side; an empty sum's zeros are no product
  const bool both = dx && dw && any;
  if (dx && M > 0)
    if (const cudaError_t e = product(Product::kNnTiles, rows.codes, ldn, rows.scales, w_codes, w_code_stride, w_scales, dx, K, false, M, K, N, s, both ? kFirst : kBehind))
      return cuda_result(who, e);
  if (dw && N > 0)
    return cuda_result(who, product(Product::kTnColumns, cols.codes, ldn, cols.scales, xcols.codes, ldk, xcols.scales, dw, K, false, N, K, M, s, both ? kBeside : kBehind));
  return 0;
}

int flame_fp8_product_faults(unsigned int* count) {
  const char* who = "flame_fp8_product_faults";
  if (!count) return refuse(who, "null count");
  // a copy on the default stream would not wait for streams that do not synchronise with it
  if (const cudaError_t e = cudaDeviceSynchronize()) return cuda_result(who, e);
  return cuda_result(who, cudaMemcpyFromSymbol(count, g_wait_faults, sizeof(*count)));
}

}  // extern "C"
