// Matrix product of FP8 E4M3 operands with one fp32 scale for each block of 128, written for sm_100a, and the quantiser that
// makes such operands from BF16 matrices.
//
//   C[m][n] = sum over blocks kb of sa(m, kb) * sb(n, kb) * (sum over k in kb of a(m, k) * b(n, k))
//
// A block runs along the contraction: 1 x 128 of a row ("rows"), 128 x 1 of a column ("columns"), or 128 x 128 ("tiles", a
// weight, which then serves the product and its transpose with the same codes).
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
struct ProductArgs {
  const uint8_t* a;
  const uint8_t* b;
  const float* sa;
  const float* sb;
  size_t a_stride, b_stride;
  void* c;
  size_t c_stride;
  uint32_t M, N, K;
  uint32_t sa_stride, sb_stride;   // floats between rows of the scale arrays
};

// Simple form: a 64 x 64 tile of C for 256 threads, 4 x 4 each; 32 values of the contraction at a time in shared memory as
// binary32 numbers.
template <bool kAmn, bool kBmn, bool kBvec, typename T>
__global__ void __launch_bounds__(256) fp8_product_simple_kernel(const __grid_constant__ ProductArgs p) {
  pdl_prologue();
  __shared__ float as[32][65], bs[32][65];
  const uint32_t tiles_n = (p.N + 63) / 64;
  const uint32_t m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
  const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (uint32_t kb = 0; kb * kBlock < p.K; ++kb) {
    float part[4][4] = {};
    for (uint32_t k0 = kb * kBlock; k0 < (kb + 1) * kBlock && k0 < p.K; k0 += 32) {
      for (uint32_t i = threadIdx.x; i < 64 * 32; i += 256) {
        const uint32_t ka = kAmn ? i / 64 : i % 32, ma = kAmn ? i % 64 : i / 32;
        const uint32_t k = k0 + ka, m = m0 + ma;
        as[ka][ma] = (k < p.K && m < p.M) ? fp8_decode(p.a[kAmn ? (size_t)k * p.a_stride + m : (size_t)m * p.a_stride + k]) : 0.0f;
        const uint32_t kc = kBmn ? i / 64 : i % 32, nc = kBmn ? i % 64 : i / 32;
        const uint32_t kk = k0 + kc, n = n0 + nc;
        bs[kc][nc] = (kk < p.K && n < p.N) ? fp8_decode(p.b[kBmn ? (size_t)kk * p.b_stride + n : (size_t)n * p.b_stride + kk]) : 0.0f;
      }
      __syncthreads();
#pragma unroll 8
      for (int k = 0; k < 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[k][ty + 16 * i], bs[k][tx + 16 * j], part[i][j]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
        if (m >= p.M || n >= p.N) continue;
        const float sa = kAmn ? p.sa[(size_t)kb * p.sa_stride + m] : p.sa[(size_t)m * p.sa_stride + kb];
        const float sb = kBvec ? (kBmn ? p.sb[(size_t)kb * p.sb_stride + n] : p.sb[(size_t)n * p.sb_stride + kb])
                               : (kBmn ? p.sb[(size_t)kb * p.sb_stride + n / kBlock] : p.sb[(size_t)(n / kBlock) * p.sb_stride + kb]);
        acc[i][j] = fmaf(sa * sb, part[i][j], acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      T* c = static_cast<T*>(p.c) + (size_t)m * p.c_stride + n;
      if constexpr (sizeof(T) == 2) *c = __float2bfloat16_rn(acc[i][j]);
      else *c = acc[i][j];
    }
}

template <bool kAmn, bool kBmn, bool kBvec>
cudaError_t launch_product(const ProductArgs& p, bool f32, cudaStream_t s) {
  const uint64_t tiles = (uint64_t)((p.M + 63) / 64) * ((p.N + 63) / 64);
  if (f32) return launch_after(fp8_product_simple_kernel<kAmn, kBmn, kBvec, float>, (unsigned)tiles, 256, 0, s, p);
  return launch_after(fp8_product_simple_kernel<kAmn, kBmn, kBvec, __nv_bfloat16>, (unsigned)tiles, 256, 0, s, p);
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
  ProductArgs p;
  p.a = static_cast<const uint8_t*>(a_codes); p.b = static_cast<const uint8_t*>(b_codes);
  p.sa = static_cast<const float*>(a_scales); p.sb = static_cast<const float*>(b_scales);
  p.a_stride = a_stride; p.b_stride = b_stride; p.c = c; p.c_stride = c_stride;
  p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K;
  auto blocks_of = [](size_t n) { return (uint32_t)((n + 127) / 128); };
  p.sa_stride = tn_cols ? (uint32_t)M : blocks_of(K);
  p.sb_stride = tn_cols ? (uint32_t)N : nn_tiles ? blocks_of(N) : blocks_of(K);
  const bool f32 = c_dtype == FLAME_OFFLOAD_DTYPE_F32;
  cudaStream_t s = (cudaStream_t)stream;
  if (nt_tiles) return (int)launch_product<false, false, false>(p, f32, s);
  if (nt_rows) return (int)launch_product<false, false, true>(p, f32, s);
  if (nn_tiles) return (int)launch_product<false, true, false>(p, f32, s);
  return (int)launch_product<true, true, true>(p, f32, s);
}

}  // extern "C"
