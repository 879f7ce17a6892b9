// Matrix product of FP8 E4M3 operands with one fp32 scale for each block of 128, written for sm_100a, and the quantiser that
// makes such operands from BF16 matrices.
//
//   C[m][n] = sum over blocks kb of sa(m, kb) * sb(n, kb) * (sum over k in kb of a(m, k) * b(n, k))
//
// A block runs along the contraction: 1 x 128 of a row ("rows"), 128 x 1 of a column ("columns"), or 128 x 128 ("tiles", a
// weight, which then serves the product and its transpose with the same codes).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "codec_kernels.cuh"
#include "common.h"
#include "fp8_device.cuh"

namespace flame_b200 {
namespace {

constexpr int kBlock = 128;

// ---- quantiser ------------------------------------------------------------------
// A thread block owns a 128 x 128 tile: thread (r, c) = (t / 16, t % 16) holds columns 8c..8c+7 of rows r, r + 16, ..., r + 112
// as eight 16-byte loads, and keeps them in registers for whichever scales the caller wants: of its rows (four shuffles), of its
// columns (one shuffle and eight partial maxima through shared memory), or of the tile.  The source is read once for both.
constexpr int kQuantThreads = 256;

struct QuantArgs {
  const __nv_bfloat16* x;
  size_t x_stride;
  uint32_t rows, cols;
  uint8_t* row_codes;        // rows or tiles
  float* row_scales;
  uint8_t* col_codes;        // columns
  float* col_scales;
  size_t code_stride;
  uint32_t tiles_across;     // ceil(cols / 128)
};

// kVec: 16-byte loads (rows start on 16 bytes and cols % 8 == 0)
template <bool kVec, bool kRows, bool kCols, bool kTile>
__global__ void __launch_bounds__(kQuantThreads) fp8_quant_kernel(const __grid_constant__ QuantArgs a) {
  pdl_prologue();
  __shared__ float part[8][kBlock];
  const uint32_t tm = blockIdx.x / a.tiles_across, tn = blockIdx.x % a.tiles_across;
  const uint32_t t = threadIdx.x, lr = t >> 4, lc = t & 15;
  const uint32_t col = tn * kBlock + lc * 8;
  uint4 raw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t row = tm * kBlock + lr + 16 * j;
    raw[j] = make_uint4(0u, 0u, 0u, 0u);
    if (row < a.rows && col < a.cols) {
      const __nv_bfloat16* src = a.x + (size_t)row * a.x_stride + col;
      if (kVec) {
        raw[j] = *reinterpret_cast<const uint4*>(src);
      } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < a.cols) w[i / 2] |= (uint32_t)__bfloat16_as_ushort(src[i]) << (16 * (i & 1));
        raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  auto unpack = [&](int j, float (&f)[8]) {
    const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
  };
  auto put = [&](uint8_t* codes, int j, const uint2& c) {
    const uint32_t row = tm * kBlock + lr + 16 * j;
    if (row < a.rows && col < a.cols) *reinterpret_cast<uint2*>(codes + (size_t)row * a.code_stride + col) = c;   // the row's padding gets zeros
  };
  float cmax[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cmax[i] = 0.0f;
  float tmax = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float f[8], m = 0.0f;
    unpack(j, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = fabsf(f[i]);
      if (kRows || kTile) m = fmaxf(m, v);
      if (kCols) cmax[i] = fmaxf(cmax[i], v);
    }
    if (kTile) tmax = fmaxf(tmax, m);
    if (kRows) {
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
      float s;
      put(a.row_codes, j, fp8_encode8(f, m, s));
      const uint32_t row = tm * kBlock + lr + 16 * j;
      if (lc == 0 && row < a.rows) a.row_scales[(size_t)row * a.tiles_across + tn] = s;
    }
  }
  if (kTile) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xFFFFFFFFu, tmax, d));
    if ((t & 31) == 0) part[0][t >> 5] = tmax;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) tmax = fmaxf(tmax, part[0][k]);
    const Fp8Scale s = fp8_scale_of(tmax);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f[8];
      unpack(j, f);
      put(a.row_codes, j, fp8_encode8(f, s));
    }
    if (t == 0) a.row_scales[(size_t)tm * a.tiles_across + tn] = s.scale;
  }
  if (kCols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cmax[i] = fmaxf(cmax[i], __shfl_xor_sync(0xFFFFFFFFu, cmax[i], 16));
    if ((t & 16) == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[t >> 5][lc * 8 + i] = cmax[i];
    }
    __syncthreads();
    Fp8Scale s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float m = part[0][lc * 8 + i];
#pragma unroll
      for (int k = 1; k < 8; ++k) m = fmaxf(m, part[k][lc * 8 + i]);
      s[i] = fp8_scale_of(m);
    }
    if (lr == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < a.cols) a.col_scales[(size_t)tm * a.cols + col + i] = s[i].scale;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f[8];
      unpack(j, f);
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = fp8_encode2(fp8_scaled(f[2 * i], s[2 * i]), fp8_scaled(f[2 * i + 1], s[2 * i + 1]));
      put(a.col_codes, j, make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16)));
    }
  }
}

// ---- codes back to numbers ---------------------------------------------------------
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
  const size_t total = (size_t)a.rows * across;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(i / across), c0 = (uint32_t)(i - (size_t)row * across) * 8;
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
    T* out = static_cast<T*>(a.out) + (size_t)row * a.cols + c0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c0 + k < a.cols) {
        const float v = fp8_decode(((k < 4 ? w.x : w.y) >> (8 * (k & 3))) & 0xFFu) * s[(c0 + k) / a.across];
        if constexpr (sizeof(T) == 2) out[k] = __float2bfloat16_rn(v);
        else out[k] = v;
      }
  }
}

// ---- product ------------------------------------------------------------------------
// One pass over the contraction in blocks of 128.  Roles of a thread block (11 warps):
//   warps 0-7  epilogue: per block of the contraction they read the tensor cores' sums from tensor memory (32 rows x BN/2 columns a
//              warp, a thread is a row) and add them to fp32 registers with the block's scales;
//   warp 8     copies tiles of both operands to shared memory (TMA, 128-byte swizzle, out-of-range elements are zeros);
//   warp 9     issues tcgen05.mma kind::f8f6f4, four of them (32 deep each) for a block of 128, into one of two accumulators;
//   warp 10    fetches the block's scales, one block ahead, and puts them into shared memory.
// Operands lie in shared memory as they lie in global memory: along the contraction (K-major) or along the rows of C (MN-major,
// the weight of the input gradient and both operands of the weight gradient), which the matrix descriptor says; nothing is
// transposed.  A block's sum is scaled by one fused multiply-add a number, which is why each block needs an accumulator of its own
// in tensor memory: two take turns, so that the tensor cores work on one while the other is read.
//
// Few tiles (serving, one token): a cluster of up to eight thread blocks shares a tile of C, each takes a range of the
// contraction, and their sums are joined through distributed shared memory in the order of the ranks.
//
// Every wait gives up after two seconds: the kernel then counts the fault (flame_fp8_product_faults), waits for its own copies and
// returns its tensor memory.
constexpr int kEpiWarps = 8;
constexpr int kProductThreads = 32 * (kEpiWarps + 4);
constexpr int kTileM = 128;
constexpr int kStagePitch = 80;                 // bytes from row to row of a warp's output staging: 64 and 16 against bank conflicts
constexpr int kStageBytes = 32 * kStagePitch;

__device__ unsigned int g_wait_faults;

struct ProductArgs {
  const float* sa;
  const float* sb;
  void* c;
  size_t c_stride;
  uint32_t M, N, K;
  uint32_t sa_stride, sb_stride;   // floats between rows of the scale arrays
  uint32_t tiles_m, tiles_n, blocks_k;
  uint32_t vec;                    // rows of C start on 16 bytes
};

template <int BN, int STAGES>
struct ProductSmem {
  static constexpr int kA = kTileM * kBlock, kB = BN * kBlock, kStage = kA + kB;
  static constexpr int kScales = (kTileM + BN) * 4;                  // of one block of the contraction
  static constexpr int kOffScales = STAGES * kStage;
  static constexpr int kOffStaging = kOffScales + 2 * kScales;
  static constexpr int kOffBars = kOffStaging + kEpiWarps * kStageBytes;
  static constexpr int kBytes = kOffBars + 256 + 1024;               // and room to start on 1024 bytes
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ uint64_t clock_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// false: two seconds have passed
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  uint64_t since = 0;
  for (uint32_t n = 0;; ++n) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((n & 255u) == 255u) {
      const uint64_t now = clock_ns();
      if (since == 0) since = now;
      else if (now - since > 2000000000ull) { atomicAdd(&g_wait_faults, 1u); return false; }
    }
  }
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
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
__device__ __forceinline__ void mma_fp8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }"
               ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// The wait belongs to the same statement: nothing else tells the compiler that the registers are not there before it.
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                 "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
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
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 peer_load4(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
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
__device__ __forceinline__ void to_bytes16(const float* v, uint4& o) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    o = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
}

template <bool kAmn, bool kBmn, bool kBvec, int BN, int STAGES, typename T>
__global__ void __launch_bounds__(kProductThreads, 1)
fp8_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ ProductArgs p) {
  using S = ProductSmem<BN, STAGES>;
  constexpr int kHalf = BN / 2;                                  // columns of an epilogue warp
  constexpr uint32_t kTmemCols = 2 * BN;
  // D fp32, A and B e4m3, major-ness, N / 8, M / 16
  constexpr uint32_t kIdesc = (1u << 4) | (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) | ((uint32_t)(BN / 8) << 17) | ((uint32_t)(kTileM / 16) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  const uint32_t base = smem_addr(smem);
  const uint32_t bars = base + S::kOffBars;
  auto full = [&](uint32_t s) { return bars + 8 * s; };
  auto empty = [&](uint32_t s) { return bars + 8 * (STAGES + s); };
  auto acc_full = [&](uint32_t b) { return bars + 8 * (2 * STAGES + b); };
  auto acc_empty = [&](uint32_t b) { return bars + 8 * (2 * STAGES + 2 + b); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kOffBars + 8 * (2 * STAGES + 4));

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t splits = BN == 128 ? cluster_size() : 1, rank = BN == 128 ? cluster_rank() : 0;   // the large tile is never split
  const uint32_t worker = blockIdx.x / splits, workers = gridDim.x / splits;
  const uint32_t tiles = p.tiles_m * p.tiles_n;
  const uint32_t kb0 = (uint32_t)((uint64_t)p.blocks_k * rank / splits), kb1 = (uint32_t)((uint64_t)p.blocks_k * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < STAGES; ++s) { bar_init(full(s), 1); bar_init(empty(s), 1); }
    for (uint32_t b = 0; b < 2; ++b) { bar_init(acc_full(b), 2); bar_init(acc_empty(b), kEpiWarps); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_prologue();

  // The epilogue's sums need more registers than an equal share: 384 threads start with 168 each, 64,512 together; four warps go
  // down to 88 and eight up to 208, 64,512 again.
  if (warp < kEpiWarps) {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const uint32_t quarter = warp & 3, half = warp >> 2;
    const uint32_t row = quarter * 32 + lane;
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t t = worker; ok && t < tiles; t += workers) {
      uint32_t tm, tn;
      tile_at(p, t, tm, tn);
      const uint32_t m0 = tm * kTileM + quarter * 32;
      const uint32_t n0 = tn * BN + half * kHalf;
      const bool rows_live = m0 < p.M && n0 < p.N;
      uint64_t acc[kHalf / 2];
#pragma unroll
      for (int i = 0; i < kHalf / 2; ++i) acc[i] = 0ull;
      for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t b = it & 1;
        if (!(ok = __all_sync(0xFFFFFFFFu, bar_wait(acc_full(b), (it >> 1) & 1)))) break;   // one answer for the warp
        if (rows_live) {
          tmem_fence_after();
          const float* sc = reinterpret_cast<const float*>(smem + S::kOffScales + b * S::kScales);
          const float sa = sc[row];
          const uint32_t src = tmem + b * BN + half * kHalf + (quarter << 21);   // lane 32 * quarter in the upper 16 bits
          uint64_t s2 = 0;
          if (kBvec) s2 = pack2(__float_as_uint(sa), __float_as_uint(sa));
#pragma unroll
          for (int c = 0; c < kHalf; c += 32) {
            if (!kBvec && c % kBlock == 0) {
              const uint32_t w = __float_as_uint(sa * sc[kTileM + (half * kHalf + c) / kBlock]);
              s2 = pack2(w, w);
            }
            uint32_t v[32];
            tmem_load32(v, src + c);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              uint64_t x0 = pack2(v[2 * i], v[2 * i + 1]), x1 = pack2(v[2 * i + 2], v[2 * i + 3]);
              if (kBvec) {
                const uint4 w = *reinterpret_cast<const uint4*>(sc + kTileM + half * kHalf + c + 2 * i);
                x0 = mul2(x0, pack2(w.x, w.y));
                x1 = mul2(x1, pack2(w.z, w.w));
              }
              acc[c / 2 + i] = fma2(x0, s2, acc[c / 2 + i]);
              acc[c / 2 + i + 1] = fma2(x1, s2, acc[c / 2 + i + 1]);
            }
          }
          tmem_fence_before();
        }
        __syncwarp();
        if (lane == 0) bar_arrive(acc_empty(b));
      }
      if (BN != 128 || splits == 1) {
        if (!rows_live || !ok) continue;
        // 64 bytes of each of the warp's 32 rows at a time go through shared memory, so that neighbouring lanes write neighbouring columns
        constexpr int kCols = 64 / sizeof(T), kPer = 16 / sizeof(T);
        uint8_t* st = smem + S::kOffStaging + warp * kStageBytes;
        const uint32_t rows = p.M - m0 < 32 ? p.M - m0 : 32;
#pragma unroll
        for (int c = 0; c < kHalf; c += kCols) {
          if (n0 + c >= p.N) break;
          float f[kCols];
#pragma unroll
          for (int i = 0; i < kCols / 2; ++i) { const float2 u = unpack2(acc[c / 2 + i]); f[2 * i] = u.x; f[2 * i + 1] = u.y; }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 o;
            to_bytes16<T>(f + j * kPer, o);
            *reinterpret_cast<uint4*>(st + lane * kStagePitch + 16 * j) = o;
          }
          __syncwarp();
          T* out = static_cast<T*>(p.c) + (size_t)m0 * p.c_stride + n0 + c;
          const uint32_t cols = p.N - (n0 + c) < (uint32_t)kCols ? p.N - (n0 + c) : kCols;
          if (p.vec && cols == (uint32_t)kCols) {
#pragma unroll
            for (int r8 = 0; r8 < 32; r8 += 8) {
              const uint32_t r = r8 + lane / 4, j = lane % 4;
              if (r < rows) *reinterpret_cast<uint4*>(out + (size_t)r * p.c_stride + j * kPer) = *reinterpret_cast<const uint4*>(st + r * kStagePitch + 16 * j);
            }
          } else {
            constexpr uint32_t kRowsAtOnce = 32 / kCols;
            for (uint32_t r = lane / kCols; r < rows; r += kRowsAtOnce) {
              const uint32_t j = lane % kCols;
              if (j < cols) out[(size_t)r * p.c_stride + j] = reinterpret_cast<const T*>(st + r * kStagePitch)[j];
            }
          }
          __syncwarp();
        }
      } else {
        // this block's share of the tile, over the pipeline's buffers: every copy has landed and every product has been read
        float* mine = reinterpret_cast<float*>(smem) + (size_t)row * (BN + 4) + half * kHalf;
        if (rows_live) {
#pragma unroll
          for (int i = 0; i < kHalf / 2; i += 2) {
            const float2 u = unpack2(acc[i]), w = unpack2(acc[i + 1]);
            *reinterpret_cast<float4*>(mine + 2 * i) = make_float4(u.x, u.y, w.x, w.y);
          }
        }
      }
    }
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = worker; ok && t < tiles; t += workers) {
          uint32_t tm, tn;
          tile_at(p, t, tm, tn);
          for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
            const uint32_t s = it % STAGES, round = it / STAGES;
            if (!(ok = bar_wait(empty(s), (round & 1) ^ 1))) break;
            bar_expect(full(s), S::kStage);
            const uint32_t sa = base + s * S::kStage, sb = sa + S::kA;
            const int32_t k = (int32_t)(kb * kBlock), m = (int32_t)(tm * kTileM), n = (int32_t)(tn * BN);
            if (kAmn) tma_load(sa, &map_a, m, k, full(s));
            else tma_load(sa, &map_a, k, m, full(s));
            if (kBmn) {
#pragma unroll
              for (int j = 0; j < BN / kBlock; ++j) tma_load(sb + j * kBlock * kBlock, &map_b, n + j * kBlock, k, full(s));
            } else {
              tma_load(sb, &map_b, k, n, full(s));
            }
          }
        }
        if (!ok)      // nothing may be in flight when the block ends
          for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i) bar_wait(full(i % STAGES), (i / STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == 9) {
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = worker; ok && t < tiles; t += workers) {
          for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
            const uint32_t s = it % STAGES, b = it & 1;
            if (!(ok = bar_wait(acc_empty(b), ((it >> 1) & 1) ^ 1))) break;
            if (!(ok = bar_wait(full(s), (it / STAGES) & 1))) break;
            tmem_fence_after();
            const uint32_t sa = base + s * S::kStage, sb = sa + S::kA;
            // 32 deep a step: 32 bytes along a K-major row, 32 rows of 128 bytes of an MN-major tile
#pragma unroll
            for (int j = 0; j < kBlock / 32; ++j)
              mma_fp8(tmem + b * BN, smem_desc<kAmn>(sa + j * (kAmn ? 32 * kBlock : 32)), smem_desc<kBmn>(sb + j * (kBmn ? 32 * kBlock : 32)), kIdesc, j > 0);
            mma_commit(empty(s));
            mma_commit(acc_full(b));
          }
        }
        if (!ok && it > 0) bar_wait(empty((it - 1) % STAGES), ((it - 1) / STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == 10) {
      uint32_t it = 0;
      bool ok = true;
      constexpr int kNb = kBvec ? BN / 32 : 1;
      for (uint32_t t = worker; ok && t < tiles; t += workers) {
        uint32_t tm, tn;
        tile_at(p, t, tm, tn);
        float a[kTileM / 32], bsc[kNb];
        auto fetch = [&](uint32_t kb) {
#pragma unroll
          for (int i = 0; i < kTileM / 32; ++i) {
            const uint32_t m = tm * kTileM + i * 32 + lane;
            a[i] = m < p.M ? __ldg(p.sa + (kAmn ? (size_t)kb * p.sa_stride + m : (size_t)m * p.sa_stride + kb)) : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < kNb; ++i) {
            if (kBvec) {
              const uint32_t n = tn * BN + i * 32 + lane;
              bsc[i] = n < p.N ? __ldg(p.sb + (kBmn ? (size_t)kb * p.sb_stride + n : (size_t)n * p.sb_stride + kb)) : 0.0f;
            } else {
              const uint32_t nb = tn * (BN / kBlock) + lane;
              bsc[i] = lane < BN / kBlock && nb * kBlock < p.N ? __ldg(p.sb + (kBmn ? (size_t)kb * p.sb_stride + nb : (size_t)nb * p.sb_stride + kb)) : 0.0f;
            }
          }
        };
        if (kb0 < kb1) fetch(kb0);
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t b = it & 1;
          if (!(ok = __all_sync(0xFFFFFFFFu, bar_wait(acc_empty(b), ((it >> 1) & 1) ^ 1)))) break;
          float* sc = reinterpret_cast<float*>(smem + S::kOffScales + b * S::kScales);
#pragma unroll
          for (int i = 0; i < kTileM / 32; ++i) sc[i * 32 + lane] = a[i];
          if (kBvec) {
#pragma unroll
            for (int i = 0; i < kNb; ++i) sc[kTileM + i * 32 + lane] = bsc[i];
          } else if (lane < BN / kBlock) {
            sc[kTileM + lane] = bsc[0];
          }
          __syncwarp();
          if (lane == 0) bar_arrive(acc_full(b));
          if (kb + 1 < kb1) fetch(kb + 1);
        }
      }
    }
  }

  __syncwarp();
  if (BN == 128 && splits > 1) {      // one tile for each cluster
    cluster_sync_all();
    if (warp < kEpiWarps && worker < tiles) {
      uint32_t tm, tn;
      tile_at(p, worker, tm, tn);
      const uint32_t rows = p.M - tm * kTileM < (uint32_t)kTileM ? p.M - tm * kTileM : kTileM;
      for (uint32_t i = rank * 256 + threadIdx.x; i < rows * (BN / 4); i += splits * 256) {
        const uint32_t r = i / (BN / 4), c = i % (BN / 4) * 4, n = tn * BN + c;
        if (n >= p.N) continue;
        const uint32_t at = base + (r * (BN + 4) + c) * 4;
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
    cluster_sync_all();   // nobody's shared memory goes away while it is read
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
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

template <bool kAmn, bool kBmn, bool kBvec, int BN, int STAGES, typename T>
cudaError_t launch_tiles(const Operands& o, ProductArgs p, uint32_t splits, uint32_t blocks, cudaStream_t stream) {
  CUtensorMap map_a, map_b;
  const bool ok = byte_matrix(&map_a, o.a, kAmn ? p.K : p.M, kAmn ? p.M : p.K, o.a_stride, kTileM) &&
                  byte_matrix(&map_b, o.b, kBmn ? p.K : p.N, kBmn ? p.N : p.K, o.b_stride, kBmn ? kBlock : BN);
  if (!ok) return cudaErrorNotSupported;
  auto kern = fp8_product_kernel<kAmn, kBmn, kBvec, BN, STAGES, T>;
  constexpr int kSmem = ProductSmem<BN, STAGES>::kBytes;
  if (const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kProductThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
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
  p.tiles_m = (p.M + kTileM - 1) / kTileM;
  p.blocks_k = (p.K + kBlock - 1) / kBlock;
  p.vec = (reinterpret_cast<uintptr_t>(p.c) & 15u) == 0 && (p.c_stride * sizeof(T)) % 16 == 0;
  p.tiles_n = (p.N + 255) / 256;
  uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n;
  if (tiles >= (uint64_t)sms) return launch_tiles<kAmn, kBmn, kBvec, 256, 4, T>(o, p, 1, (uint32_t)sms, stream);
  p.tiles_n = (p.N + 127) / 128;
  tiles = (uint64_t)p.tiles_m * p.tiles_n;
  uint32_t splits = 1;
  while (splits < 8 && tiles * splits * 2 <= (uint64_t)sms && splits * 2 <= p.blocks_k) splits *= 2;
  const uint32_t blocks = splits > 1 ? (uint32_t)tiles * splits : (uint32_t)(tiles < (uint64_t)sms ? tiles : (uint64_t)sms);
  return launch_tiles<kAmn, kBmn, kBvec, 128, 5, T>(o, p, splits, blocks, stream);
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
  if (rows > kMostSize || cols > kMostSize) return refuse(who, "matrix too large");
  if (x_stride < cols || code_stride < cols || code_stride % 16 != 0) return refuse(who, "a stride is smaller than the row, or the code stride is no multiple of 16");
  if (rows == 0 || cols == 0) return 0;
  if (!tile && !row && !col) return refuse(who, "nothing to make");
  if (!x || ((tile || row) && (!codes || !scales)) || (col && !column_scales)) return refuse(who, "null tensor");
  if (!al(x, 2) || !al(codes, 16) || !al(column_codes, 16) || !al(scales, 4) || !al(column_scales, 4)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  const uint64_t down = (rows + 127) / 128, across = (cols + 127) / 128;
  if (down * across > 0x7FFFFFFFull) return refuse(who, "matrix too large");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return (int)cudaErrorLaunchFailure;
  QuantArgs a;
  a.x = static_cast<const __nv_bfloat16*>(x); a.x_stride = x_stride; a.rows = (uint32_t)rows; a.cols = (uint32_t)cols;
  a.row_codes = static_cast<uint8_t*>(codes); a.row_scales = static_cast<float*>(scales);
  a.col_codes = static_cast<uint8_t*>(column_codes); a.col_scales = static_cast<float*>(column_scales);
  a.code_stride = code_stride; a.tiles_across = (uint32_t)across;
  const bool vec = al(x, 16) && x_stride % 8 == 0 && cols % 8 == 0;
  auto go = [&](auto kern) { return (int)launch_after(kern, (unsigned)(down * across), kQuantThreads, 0, (cudaStream_t)stream, a); };
  if (tile) return vec ? go(fp8_quant_kernel<true, false, false, true>) : go(fp8_quant_kernel<false, false, false, true>);
  if (row && col) return vec ? go(fp8_quant_kernel<true, true, true, false>) : go(fp8_quant_kernel<false, true, true, false>);
  if (row) return vec ? go(fp8_quant_kernel<true, true, false, false>) : go(fp8_quant_kernel<false, true, false, false>);
  return vec ? go(fp8_quant_kernel<true, false, true, false>) : go(fp8_quant_kernel<false, false, true, false>);
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
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return (int)cudaErrorLaunchFailure;
  DequantArgs a;
  a.codes = static_cast<const uint8_t*>(codes); a.code_stride = code_stride; a.scales = static_cast<const float*>(scales);
  a.rows = (uint32_t)rows; a.cols = (uint32_t)cols; a.out = out;
  a.down = blocks == FLAME_FP8_BLOCKS_ROWS ? 1 : kBlock;
  a.across = blocks == FLAME_FP8_BLOCKS_COLUMNS ? 1 : kBlock;
  a.scales_across = blocks == FLAME_FP8_BLOCKS_COLUMNS ? (uint32_t)cols : (uint32_t)((cols + 127) / 128);
  const uint64_t blocks_wanted = ((uint64_t)rows * ((cols + 7) / 8) + 255) / 256;
  const unsigned grid = (unsigned)(blocks_wanted < 148 * 32 ? blocks_wanted : 148 * 32);
  return out_dtype == FLAME_OFFLOAD_DTYPE_F32 ? (int)launch_after(fp8_dequant_kernel<float>, grid, 256, 0, (cudaStream_t)stream, a)
                                              : (int)launch_after(fp8_dequant_kernel<__nv_bfloat16>, grid, 256, 0, (cudaStream_t)stream, a);
}

int flame_fp8_product(const void* a_codes, size_t a_stride, const void* a_scales, int a_blocks, const void* b_codes, size_t b_stride,
                      const void* b_scales, int b_blocks, int b_transposed, void* c, size_t c_stride, int c_dtype, size_t M, size_t N, size_t K, void* stream) {
  const char* who = "flame_fp8_product";
  const bool nt_tiles = a_blocks == FLAME_FP8_BLOCKS_ROWS && b_blocks == FLAME_FP8_BLOCKS_TILES && b_transposed;
  const bool nt_rows = a_blocks == FLAME_FP8_BLOCKS_ROWS && b_blocks == FLAME_FP8_BLOCKS_ROWS && b_transposed;
  const bool nn_tiles = a_blocks == FLAME_FP8_BLOCKS_ROWS && b_blocks == FLAME_FP8_BLOCKS_TILES && !b_transposed;
  const bool tn_cols = a_blocks == FLAME_FP8_BLOCKS_COLUMNS && b_blocks == FLAME_FP8_BLOCKS_COLUMNS && !b_transposed;
  if (!nt_tiles && !nt_rows && !nn_tiles && !tn_cols)
    return refuse(who, "the blocks of both operands must run along the contraction: rows x rows^T, rows x tiles^T, rows x tiles or columns^T x columns");
  if (c_dtype != FLAME_OFFLOAD_DTYPE_BF16 && c_dtype != FLAME_OFFLOAD_DTYPE_F32) return refuse(who, "the output is BF16 or F32");
  if (M > kMostSize || N > kMostSize || K > kMostSize) return refuse(who, "matrix too large");
  const size_t a_row = tn_cols ? M : K, b_row = b_transposed ? K : N;
  if (a_stride < a_row || b_stride < b_row || a_stride % 16 != 0 || b_stride % 16 != 0 || c_stride < N) return refuse(who, "a stride is smaller than its row, or a code stride no multiple of 16");
  if (M == 0 || N == 0) return 0;
  if (!c || !al(c, c_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2)) return refuse(who, "null or misaligned output");
  if (K == 0) {   // an empty sum
    const size_t size = c_dtype == FLAME_OFFLOAD_DTYPE_F32 ? 4 : 2;
    return (int)cudaMemset2DAsync(c, c_stride * size, 0, N * size, M, (cudaStream_t)stream);
  }
  if (!a_codes || !b_codes || !a_scales || !b_scales) return refuse(who, "null tensor");
  if (!al(a_codes, 16) || !al(b_codes, 16) || !al(a_scales, 4) || !al(b_scales, 4)) return refuse(who, "misaligned tensor (codes: 16 bytes)");
  if (((M + 63) / 64) * ((N + 63) / 64) > 0x7FFFFFFFull) return refuse(who, "matrix too large");
  if (fault_fires(FLAME_OFFLOAD_FAULT_KERNEL)) return (int)cudaErrorLaunchFailure;
  const Operands o = {static_cast<const uint8_t*>(a_codes), static_cast<const uint8_t*>(b_codes), a_stride, b_stride};
  ProductArgs p = {};
  p.sa = static_cast<const float*>(a_scales); p.sb = static_cast<const float*>(b_scales);
  p.c = c; p.c_stride = c_stride;
  p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K;
  auto blocks_of = [](size_t n) { return (uint32_t)((n + 127) / 128); };
  p.sa_stride = tn_cols ? (uint32_t)M : blocks_of(K);
  p.sb_stride = tn_cols ? (uint32_t)N : nn_tiles ? blocks_of(N) : blocks_of(K);
  const bool f32 = c_dtype == FLAME_OFFLOAD_DTYPE_F32;
  cudaStream_t s = (cudaStream_t)stream;
  if (nt_tiles) return (int)launch_product<false, false, false>(o, p, f32, s);
  if (nt_rows) return (int)launch_product<false, false, true>(o, p, f32, s);
  if (nn_tiles) return (int)launch_product<false, true, false>(o, p, f32, s);
  return (int)launch_product<true, true, true>(o, p, f32, s);
}

int flame_fp8_product_faults(unsigned int* count) {
  if (!count) return (int)cudaErrorInvalidValue;
  return (int)cudaMemcpyFromSymbol(count, g_wait_faults, sizeof(*count));
}

}  // extern "C"
