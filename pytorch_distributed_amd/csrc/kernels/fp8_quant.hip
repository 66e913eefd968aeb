// Block quantisation to 8-bit floating point (OCP e4m3) for gfx950.
//
// A block of 128 values shares a power-of-two scale 2^e with
//     e = min { integer >= -127 : max|x| <= 448 * 2^e },     q = e4m3(x / 2^e), ties to even,
// stored as the byte e + 127 (the E8M0 form the block-scaled matrix instruction takes). Dividing by a
// power of two is exact, so the rounding to e4m3 is the only error: at most half a step, 2^-4 of a
// normal value. With max|x| = m 2^k (1 <= m < 2) and 448 = 1.75 * 2^8, e = k - 8, plus one when
// m > 1.75: read off the float's bits, no logarithm. An infinity or a NaN takes no part in its block's
// maximum and becomes the e4m3 NaN (0x7f / 0xff), so a product with it is NaN where bf16 would be.
//
// Three block shapes, any combination of the two outputs in ONE pass over x [R, C]:
//   rows      1 x 128 along C:  q [R, Cp],  scale [R, Sc]       (contraction over C)
//   columns   128 x 1 along R:  qt [C, Rp], scale [C, Sr]       (transposed: contraction over R)
//   tiles     128 x 128, one scale, both layouts                (weights: both contractions)
// Cp / Rp are C / R rounded up to 128 (padding: zeros), Sc / Sr the block counts rounded up to 4
// (padding: zero bytes). The column sums of x (a bias gradient) can ride along: fp32 partial sums per
// 128-row block, folded in a fixed order by fp8_gemm's last launch. Several matrices share a launch: a layer's
// small ones cost a launch, not their bytes.
//
// What bounds it: memory. A workgroup owns a 128 x 128 tile held in registers (8 rows x 8 columns per
// thread), so x is read once for both layouts; the transposed bytes pass through a swizzled 16 KiB LDS
// tile and leave as whole 128-byte lines. Measured: 65536 x 5120 bf16 to both layouts 288 us = 4.7 TB/s, 6400 x 1600
// fp32 by tiles 12.7 us = 4.8 TB/s (a large copy reaches 5.1); a small matrix costs its launch, 7 us. bf16 values stay
// packed in registers: eight workgroups on a compute unit instead of five (306 -> 288; 8192 x 5120 54 -> 46).
#include <type_traits>

#include "common.h"
#include "pda_kernels.h"

namespace pda {
namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 256;
constexpr float kInf = __builtin_inff();

// Scale byte of a block with largest finite magnitude `amax` (>= 0), from the float's exponent and
// mantissa. Subnormal magnitudes are far below 448 * 2^-127: byte 0.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased exponent - 8 = (e + 127)
  return uint32_t(max(e, 0));
}

// 2^-(byte - 127). Bytes run from 0 to 247 (the largest float, just below 2^128, takes 2^120), so the result is a normal float.
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// |x| of the finite values, 0 for the others.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < kInf ? a : 0.f;
}

// Eight values of one row, as they are kept: bf16 pairs (half the registers, so eight workgroups fit a compute unit
// where five would), or floats.
template <typename T>
struct Eight;
template <>
struct Eight<bf16_raw> {
  u32x4 w;
  __device__ __forceinline__ float operator[](int k) const { return k & 1 ? bf16_hi(w[k / 2]) : bf16_lo(w[k / 2]); }
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(w)); }  // unpacked again from here on, not held
};
template <>
struct Eight<float> {
  f32x4 a, b;
  __device__ __forceinline__ float operator[](int k) const { return k < 4 ? a[k & 3] : b[k & 3]; }
  __device__ __forceinline__ void forget() {}
};

// Eight values of one row starting at column c (c % 8 == 0); columns >= C and rows >= R read as zeros. Rows lie at
// any multiple of a value: global memory takes 16-byte accesses at any alignment (41160 x 2374 bf16 by columns, rows
// at multiples of 4 bytes: 156 us value by value, 70 so).
typedef u32x4 __attribute__((aligned(2))) u32x4_anywhere;
typedef f32x4 __attribute__((aligned(4))) f32x4_anywhere;
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* __restrict__ x, int64_t ld, int R, int C, int row, int c) {
  Eight<T> v;
  if constexpr (sizeof(T) == 2) v.w = u32x4{0u, 0u, 0u, 0u};
  else v.a = v.b = f32x4{0.f, 0.f, 0.f, 0.f};
  if (row >= R || c >= C) return v;
  const T* p = x + int64_t(row) * ld + c;
  if (c + 8 <= C) {
    if constexpr (sizeof(T) == 2) {
      v.w = *reinterpret_cast<const u32x4_anywhere*>(p);
    } else {
      v.a = *reinterpret_cast<const f32x4_anywhere*>(p);
      v.b = *reinterpret_cast<const f32x4_anywhere*>(p + 4);
    }
    return v;
  }
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (c + i < C) {
      if constexpr (sizeof(T) == 2) v.w[i / 2] |= uint32_t(p[i]) << (16 * (i & 1));
      else if (i < 4) v.a[i] = p[i];
      else v.b[i - 4] = p[i];
    }
  return v;
}

// Maximum over the 16 lanes of a row group, by rotations inside it.
__device__ __forceinline__ float max16(float m) {
  auto turned = [](float x, auto by) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + decltype(by)::value, 0xf, 0xf, false));
  };
  m = fmaxf(m, turned(m, std::integral_constant<int, 8>{}));
  m = fmaxf(m, turned(m, std::integral_constant<int, 4>{}));
  m = fmaxf(m, turned(m, std::integral_constant<int, 2>{}));
  return fmaxf(m, turned(m, std::integral_constant<int, 1>{}));
}

// Thread (g = tid / 16, j = tid % 16) holds rows 8 g .. 8 g + 7 and columns 8 j .. 8 j + 7 of the tile.
struct Matrix {
  const void* x;
  int64_t ld;
  int R, C, blocks;
  bool tiles;
  uint8_t *q, *s, *qt, *st;  // null: not wanted
  float* sums;
};
struct Matrices {
  Matrix m[3];
};

template <typename T>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 8 : 5))) void quantize_kernel(const Matrices all) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[kBlock * kBlock];
  __shared__ float red[4][kBlock];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = tid >> 4, j = tid & 15;
  int block = blockIdx.x, which = 0;
  while (block >= all.m[which].blocks) block -= all.m[which++].blocks;  // (the blocks' sum is the grid)
  const Matrix& mat = all.m[which];
  const T* __restrict__ x = (const T*)mat.x;
  const int R = mat.R, C = mat.C;
  const int n_cb = (C + kBlock - 1) / kBlock, n_rb = (R + kBlock - 1) / kBlock;
  const int rb = block / n_cb, cb = block - rb * n_cb;
  const int row0 = rb * kBlock + 8 * g, col0 = cb * kBlock + 8 * j;
  uint8_t *const q = mat.q, *const s = mat.s, *const qt = mat.qt, *const st = mat.st;

  Eight<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = load8<T>(x, mat.ld, R, C, row0 + i, col0);

  float tile_inv = 1.f;
  uint32_t tile_byte = 0;
  if (mat.tiles) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[i][k]));
    m = block_max<kThreads>(m, &red[0][0]);
    tile_byte = scale_byte(m);
    tile_inv = inverse_scale(tile_byte);
    // one byte per tile in each orientation; the last tile of a row of tiles also clears the padding
    if (tid == 0) {
      if (q) {
        const int pitch = (n_cb + 3) & ~3;
        s[int64_t(rb) * pitch + cb] = uint8_t(tile_byte);
        if (cb == n_cb - 1)
          for (int k = n_cb; k < pitch; ++k) s[int64_t(rb) * pitch + k] = 0;
      }
      if (qt) {
        const int pitch = (n_rb + 3) & ~3;
        st[int64_t(cb) * pitch + rb] = uint8_t(tile_byte);
        if (rb == n_rb - 1)
          for (int k = n_rb; k < pitch; ++k) st[int64_t(cb) * pitch + k] = 0;
      }
    }
  }

  auto forget = [&]() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].forget();
  };
  forget();
  if (q) {
    const int64_t Cp = int64_t(n_cb) * kBlock;
    const int pitch = (n_cb + 3) & ~3;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + i;
      float inv = tile_inv;
      if (!mat.tiles) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[i][k]));
        m = max16(m);
        const uint32_t byte = scale_byte(m);
        inv = inverse_scale(byte);
        if (row < R && j == 0) {
          s[int64_t(row) * pitch + cb] = uint8_t(byte);
          if (cb == n_cb - 1)
            for (int k = n_cb; k < pitch; ++k) s[int64_t(row) * pitch + k] = 0;
        }
      }
      if (row < R) {
        u32x2 w = {pack_fp8x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                   pack_fp8x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv)};
        *reinterpret_cast<u32x2*>(q + int64_t(row) * Cp + col0) = w;
      }
    }
  }

  forget();
  if (mat.sums) {  // column sums of this 128-row block: rows in a thread, row groups in a wave, waves in order
    float sum[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      sum[k] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[k] += v[i][k];
      sum[k] += __shfl_xor(sum[k], 16, 64);
      sum[k] += __shfl_xor(sum[k], 32, 64);
    }
    if (lane < 16)
#pragma unroll
      for (int k = 0; k < 8; ++k) red[wave][8 * j + k] = sum[k];
    __syncthreads();
    if (tid < kBlock && cb * kBlock + tid < C)
      mat.sums[int64_t(rb) * C + cb * kBlock + tid] = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
    __syncthreads();
  }

  forget();
  if (qt) {
    float inv[8];
    if (mat.tiles) {
#pragma unroll
      for (int k = 0; k < 8; ++k) inv[k] = tile_inv;
    } else {
      float m[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m[k] = fmaxf(m[k], finite_abs(v[i][k]));
        m[k] = fmaxf(m[k], __shfl_xor(m[k], 16, 64));
        m[k] = fmaxf(m[k], __shfl_xor(m[k], 32, 64));
      }
      if (lane < 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) red[wave][8 * j + k] = m[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = 8 * j + k;
        const uint32_t byte = scale_byte(fmaxf(fmaxf(red[0][c], red[1][c]), fmaxf(red[2][c], red[3][c])));
        inv[k] = inverse_scale(byte);
        if (g == 0 && col0 + k < C) {
          const int pitch = (n_rb + 3) & ~3;
          uint8_t* dst = st + int64_t(col0 + k) * pitch;
          dst[rb] = uint8_t(byte);
          if (rb == n_rb - 1)
            for (int b = n_rb; b < pitch; ++b) dst[b] = 0;
        }
      }
    }
    forget();
    // Column c of the tile is a 128-byte LDS row; its 16-byte chunks are permuted by the column group j
    // (the lanes of a store share the column within their group), so 8 column groups take 8 chunks.
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u32x2 w = {pack_fp8x4(v[0][k] * inv[k], v[1][k] * inv[k], v[2][k] * inv[k], v[3][k] * inv[k]),
                 pack_fp8x4(v[4][k] * inv[k], v[5][k] * inv[k], v[6][k] * inv[k], v[7][k] * inv[k])};
      const int chunk = (g >> 1) ^ (j & 7);
      *reinterpret_cast<u32x2*>(&tile[(8 * j + k) * kBlock + chunk * 16 + (g & 1) * 8]) = w;
    }
    __syncthreads();
    const int64_t Rp = int64_t(n_rb) * kBlock;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = i * 32 + (tid >> 3), chunk = tid & 7;  // 8 lanes write one 128-byte line
      const u32x4 w = *reinterpret_cast<const u32x4*>(&tile[c * kBlock + (chunk ^ ((c >> 3) & 7)) * 16]);
      const int col = cb * kBlock + c;
      if (col < C) *reinterpret_cast<u32x4*>(qt + int64_t(col) * Rp + int64_t(rb) * kBlock + chunk * 16) = w;
    }
  }
}

}  // namespace

void fp8_quantize(DType dtype, const Fp8QuantProblem* problems, int n, hipStream_t stream) {
  Matrices all = {};
  int64_t blocks = 0;
  for (int i = 0; i < n; ++i) {
    const Fp8QuantProblem& p = problems[i];
    const int64_t b = ceil_div(p.C, kBlock) * ceil_div(p.R, kBlock);
    all.m[i] = Matrix{p.x, p.ld, p.R, p.C, (int)b, p.tiles, p.q, p.scale, p.qt, p.scale_t, p.column_sums};
    blocks += b;
  }
  const dim3 grid((unsigned)blocks), block(kThreads);
  if (dtype == kBF16) hipLaunchKernelGGL(quantize_kernel<bf16_raw>, grid, block, 0, stream, all);
  else hipLaunchKernelGGL(quantize_kernel<float>, grid, block, 0, stream, all);
}

}  // namespace pda
