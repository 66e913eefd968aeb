// Block-scaled 8-bit matrix product for gfx950:
//   out[M, N] = (bias[N] +) sum_k 2^(ex[m, k/128] + ew[n, k/128]) x[m, k] w[n, k],   x, w e4m3, fp32 accumulation.
//
// Both operands are contraction-contiguous, rows padded with zeros to a multiple of 128 values; the
// scales are bytes e + 127, one per 128 values of a row or per 128 x 128 tile. v_mfma_scale_f32_32x32x64
// takes such a byte per row and applies it inside the instruction, so a block-scaled product costs no
// vector instruction per product more than an unscaled one.
//
// Structure. A workgroup of 4 waves (2 x 2) owns a square output tile, each wave a quarter as kWB x kWB
// blocks of 32 x 32. A pipeline stage is 64 values of the contraction: [tile rows][64 bytes] of each
// operand, moved global -> LDS by global_load_lds into a ring of four. The body of stage t
//   * waits until stage t + 1 has landed (counted: two younger stages stay in flight) and meets the
//     other waves, who by then have read stage t out of LDS;
//   * issues the products of stage t from registers, and between them the LDS reads of stage t + 1 and
//     the loads of stage t + 4 into the slot that stage t has left.
// One barrier per 16 matrix instructions (1,024 matrix cycles) of a wave at kWB = 4.
// The 16-byte chunk index of an LDS row is XOR-permuted with bits 2-3 of the row (on the source address:
// the destination of such a load is linear), which makes the ds_read_b128 of 32 rows conflict free. A
// lane's 32 bytes are chunks h and 2 + h of the row: the same order for both operands, and inside one
// scale block, so the instruction's own order of the contraction does not matter.
// The product is formed transposed (features on the accumulator registers, tokens on the lanes), so a
// register quad is four consecutive features of one token.
//
// fp32 results. The 8-bit matrix instructions align the 64 products of a call to the largest of them and drop
// bits: measured (random e4m3 operands) up to 1.3e-4 of sum |x w|, 5e-5 in norm, whatever the contraction's
// length. Next to a bf16 result's rounding (1.7e-3) that is nothing; an fp32 result is computed with kWide
// instead: fragments widened to bf16 on the way to v_mfma_f32_32x32x16_bf16, scale included (exact), whose
// sums are good to 6e-8, at half the matrix rate.
//
// Few output tiles (weight gradients, few tokens): the contraction is cut into slices of whole 512-value
// scale groups, fp32 partial tiles are folded in slice order by a second kernel (deterministic).
#include "attention_common.h"
#include "pda_kernels.h"

namespace pda {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;

constexpr int kThreads = 256;
constexpr int kStages = 4;
constexpr int kStageK = 64;                 // values (bytes) of the contraction per stage
constexpr int kGroupStages = 8;             // stages whose scales are fetched together: 4 blocks of 128, a dword a row
constexpr int kGroupM = 4;                  // token tiles walked together by consecutive tasks

__device__ __forceinline__ unsigned lds_addr(const char* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// LDS reads through inline assembly: the compiler would wait for all global_load_lds in flight before an
// ordinary LDS read. Completion is awaited by the stage body before the values are used.
template <int kOff>
__device__ __forceinline__ u32x4 chunk_read(unsigned addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(kOff));
  return v;
}

// Loads to LDS in buffer form: wave-uniform base and offset along the contraction in scalar registers, one
// 32-bit lane offset, and a hardware bound on the operand's bytes.
typedef __attribute__((address_space(3))) void lds_ptr_t;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bounded(const uint8_t* base, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ void load_to_lds16(__amdgpu_buffer_rsrc_t src, unsigned lane_off, unsigned off, char* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr_t*)dst, 16, (int)lane_off, (int)off, 0, 0);
}
__device__ __forceinline__ void load_to_lds4(__amdgpu_buffer_rsrc_t src, unsigned lane_off, unsigned off, char* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr_t*)dst, 4, (int)lane_off, (int)off, 0, 0);
}

__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

__device__ __forceinline__ f32x16 mfma_scaled(i32x8 a, i32x8 b, f32x16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}

// Two of the e4m3 values of `v` (its lower or upper half) times 2^(byte - 127) as bf16: exact, e4m3 has 4
// significant bits and bf16 its scale's range.
template <bool kHigh>
__device__ __forceinline__ uint32_t widen2(uint32_t v, uint32_t byte) {
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, __uint_as_float(byte << 23), kHigh);
  return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi, uint32_t byte) {
  return __builtin_bit_cast(bf16x8, u32x4{widen2<false>(lo, byte), widen2<true>(lo, byte), widen2<false>(hi, byte), widen2<true>(hi, byte)});
}

// One operand of the product: `rows` rows of `ld` bytes, scales at row >> shift.
struct Operand {
  const uint8_t* q;
  const uint8_t* scale;
  int64_t ld, ld_scale;
  int rows, shift;
};

struct Output {
  void* ptr;         // [M, N] (bf16 or fp32), or the fp32 partials [slices][M][N]
  const void* bias;  // [N] or null
  int64_t ld;
  bool bias_f32, accumulate, vec;  // vec: rows are aligned for four-value stores
};

template <int kWB, typename Out, bool kWide>
__global__ __launch_bounds__(kThreads) void fp8_gemm_kernel(Operand X, Operand W, Output O, int steps_total,
                                                            int steps_per_slice) {
  constexpr int kTile = 64 * kWB;
  constexpr int kSlab = kTile * kStageK;       // bytes of one operand's stage
  constexpr int kStageBytes = 2 * kSlab;
  constexpr int kPieces = kTile / 64;          // 16-row loads per wave, stage and operand
  constexpr int kScaleLoads = kTile / 128;     // 64-row scale loads per wave and group (both operands)
  constexpr int kScaleBytes = 2 * kTile * 4;   // one group's scales: X rows, then W rows
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* scale_smem = smem + kStages * kStageBytes;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave >> 1, wj = wave & 1;
  const int r = lane & 31, h = lane >> 5;
  const int M = X.rows, N = W.rows;

  // Tasks are dealt to the 8 XCDs in contiguous ranges; consecutive tasks walk kGroupM token tiles x all
  // feature tiles, so the workgroups of an XCD share operand rows in its L2.
  const int tiles_m = (M + kTile - 1) / kTile, tiles_n = (N + kTile - 1) / kTile;
  const int n_tiles = tiles_m * tiles_n;
  const int n_tasks = gridDim.x;
  const int q8 = n_tasks / 8, r8 = n_tasks % 8;
  const int xcd = blockIdx.x % 8, within = blockIdx.x / 8;
  const int task = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + within;
  const int slice = task / n_tiles;
  const int tile = task - slice * n_tiles;
  const int group = tile / (kGroupM * tiles_n);
  const int in_group = tile - group * (kGroupM * tiles_n);
  const int group_rows = min(kGroupM, tiles_m - group * kGroupM);
  const int m0 = (group * kGroupM + in_group % group_rows) * kTile;
  const int n0 = (in_group / group_rows) * kTile;
  const int first = slice * steps_per_slice;  // a multiple of kGroupStages
  const int n_steps = min(steps_per_slice, steps_total - first);

  // ---- staging: piece i of a slab = rows (kTile / 4) wave + 16 i .. +15, lane p -> row + p / 4, slot p % 4.
  // Rows past the end repeat the last one (never stored).
  // (All offsets fit 32 bits: a tile's rows span at most 256 * 2^22 bytes, a bound the host checks.)
  const int x_rows = min(M - m0, kTile), w_rows = min(N - n0, kTile);
  const unsigned k_bytes = (unsigned)n_steps * kStageK;
  const auto x_src = bounded(X.q + int64_t(m0) * X.ld + int64_t(first) * kStageK, (unsigned)(x_rows - 1) * (unsigned)X.ld + k_bytes);
  const auto w_src = bounded(W.q + int64_t(n0) * W.ld + int64_t(first) * kStageK, (unsigned)(w_rows - 1) * (unsigned)W.ld + k_bytes);
  unsigned x_off[kPieces], w_off[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int row = (kTile / 4) * wave + 16 * i + (lane >> 2);
    const unsigned chunk = (unsigned)(((lane & 3) ^ ((row >> 2) & 3)) * 16);
    x_off[i] = (unsigned)min(row, x_rows - 1) * (unsigned)X.ld + chunk;
    w_off[i] = (unsigned)min(row, w_rows - 1) * (unsigned)W.ld + chunk;
  }
  auto issue_one = [&](int t, int slot, int i) {  // i < 2 kPieces
    const unsigned ko = (unsigned)min(t, n_steps - 1) * kStageK;  // past the end: the last stage again (never used)
    char* dst = smem + slot * kStageBytes + ((kTile / 4) * wave + 16 * (i % kPieces)) * kStageK;
    if (i < kPieces) load_to_lds16(x_src, x_off[i], ko, dst);
    else load_to_lds16(w_src, w_off[i - kPieces], ko, dst + kSlab);
  };
  // ---- scales: group g = blocks 4 g .. 4 g + 3, a dword per row; 64 rows per load, all of one operand.
  const int n_groups = (n_steps + kGroupStages - 1) / kGroupStages;
  const bool s_of_x = wave < 2;  // waves 0, 1 fetch the scales of X's rows, waves 2, 3 those of W's
  const Operand& s_op = s_of_x ? X : W;
  const int s_row0 = s_of_x ? m0 : n0, s_last = (s_of_x ? M : N) - 1;
  const int s_lo = s_row0 >> s_op.shift, s_hi = min(s_row0 + kTile - 1, s_last) >> s_op.shift;
  const auto s_src = bounded(s_op.scale + int64_t(s_lo) * s_op.ld_scale + first / 2,
                             (unsigned)(s_hi - s_lo) * (unsigned)s_op.ld_scale + 4u * (unsigned)n_groups);
  unsigned s_off[kScaleLoads];
#pragma unroll
  for (int i = 0; i < kScaleLoads; ++i) {
    const int row = ((wave & 1) * kScaleLoads + i) * 64 + lane;
    s_off[i] = (unsigned)((min(s_row0 + row, s_last) >> s_op.shift) - s_lo) * (unsigned)s_op.ld_scale;
  }
  auto issue_scales = [&](int g) {
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i)
      load_to_lds4(s_src, s_off[i], 4u * (unsigned)min(g, n_groups - 1),
                   scale_smem + (g & 1) * kScaleBytes + (wave * kScaleLoads + i) * 256);
  };

  f32x16 acc[kWB][kWB];
#pragma unroll
  for (int a = 0; a < kWB; ++a)
#pragma unroll
    for (int b = 0; b < kWB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;

  // ---- fragment addresses: lane (r, h) reads chunks h and 2 + h of row r of each 32-row block
  const unsigned smem_base = lds_addr(smem);
  const int f = (r >> 2) & 3;
  const unsigned c0 = (unsigned)((h ^ f) << 4), c1 = (unsigned)(((2 + h) ^ f) << 4);
  const unsigned x_row = (unsigned)((32 * kWB * wi + r) * kStageK);
  const unsigned w_row = (unsigned)(kSlab + (32 * kWB * wj + r) * kStageK);
  u32x4 xf[2][kWB][2], wf[2][kWB][2];
  // read i (0 .. 4 kWB - 1) of the fragments of the stage in `slot`: w0 x0 w1 x1 ..., two chunks each
  auto frag = [&](int buf, int slot, int i) {
    const unsigned base = smem_base + slot * kStageBytes;
    const int blk = i >> 2;
    const unsigned at = base + ((i & 2) ? x_row : w_row) + ((i & 1) ? c1 : c0);
    u32x4& dst = (i & 2) ? xf[buf][blk][i & 1] : wf[buf][blk][i & 1];
    if (blk == 0) dst = chunk_read<0>(at);
    if (blk == 1) dst = chunk_read<2048>(at);
    if (blk == 2) dst = chunk_read<4096>(at);
    if (blk == 3) dst = chunk_read<6144>(at);
  };
  // the values read by `frag` exist after this point (ties every register to the wait)
  auto await_frags = [&](int buf) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int b = 0; b < kWB; ++b)
      asm volatile("" : "+v"(xf[buf][b][0]), "+v"(xf[buf][b][1]), "+v"(wf[buf][b][0]), "+v"(wf[buf][b][1]));
  };
  // scale bytes of block c (a pair of stages), read 0 .. 2 kWB - 1: X's and W's of each 32-row block in turn
  const unsigned scale_base = lds_addr(scale_smem);
  const unsigned xs_row = (unsigned)((32 * kWB * wi + r) * 4), ws_row = (unsigned)((kTile + 32 * kWB * wj + r) * 4);
  uint32_t xs[kWB], ws[kWB], xs_next[kWB], ws_next[kWB];
  auto read_scale = [&](int c, int i) {
    const unsigned at = scale_base + ((c >> 2) & 1) * kScaleBytes + (c & 3) + ((i & 1) ? ws_row : xs_row);
    uint32_t& dst = (i & 1) ? ws_next[i >> 1] : xs_next[i >> 1];
    if ((i >> 1) == 0) asm volatile("ds_read_u8 %0, %1" : "=v"(dst) : "v"(at));
    if ((i >> 1) == 1) asm volatile("ds_read_u8 %0, %1 offset:128" : "=v"(dst) : "v"(at));
    if ((i >> 1) == 2) asm volatile("ds_read_u8 %0, %1 offset:256" : "=v"(dst) : "v"(at));
    if ((i >> 1) == 3) asm volatile("ds_read_u8 %0, %1 offset:384" : "=v"(dst) : "v"(at));
  };
  auto take_scales = [&]() {  // after await_frags
#pragma unroll
    for (int b = 0; b < kWB; ++b) {
      asm volatile("" : "+v"(xs_next[b]), "+v"(ws_next[b]));
      xs[b] = xs_next[b];
      ws[b] = ws_next[b];
    }
  };
  constexpr int kLoads = 2 * kPieces;  // per wave and stage

  issue_scales(0);
#pragma unroll
  for (int t = 0; t < kStages; ++t)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) issue_one(t, t, i);
  if constexpr (kWB == 4) asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 2 * kWB; ++i) read_scale(0, i);
#pragma unroll
  for (int i = 0; i < 4 * kWB; ++i) frag(0, 0, i);
  await_frags(0);
  take_scales();

  int slot = 0;  // of stage t
  for (int t = 0; t < n_steps; t += 2) {  // n_steps is even; a pair of stages is one scale block
    if ((t & (kGroupStages - 1)) == 0) issue_scales(t / kGroupStages + 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // Stage t + u + 1 has landed (two younger stages may be in flight; a scale load among them makes the
      // count strict by that much); after the barrier everyone's part has, and nobody reads this slot any more.
      if constexpr (kWB == 4) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      const int next = (slot + 1) & (kStages - 1);
      constexpr int kProducts = kWB * kWB;
      int reads = 0, loads = 0, scales = 0;
      [[maybe_unused]] bf16x8 xb[4], wb[kWide ? kWB : 1][4];
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        const int a = i / kWB, b = i % kWB;
        if constexpr (kWide) {
          if (b == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) xb[k] = widen8(xf[u][a][k >> 1][2 * (k & 1)], xf[u][a][k >> 1][2 * (k & 1) + 1], xs[a]);
          }
          if (a == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) wb[b][k] = widen8(wf[u][b][k >> 1][2 * (k & 1)], wf[u][b][k >> 1][2 * (k & 1) + 1], ws[b]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[a][b] = attn::mfma32(wb[b][k], xb[k], acc[a][b]);
        } else {
          acc[a][b] = mfma_scaled(join(wf[u][b][0], wf[u][b][1]), join(xf[u][a][0], xf[u][a][1]), acc[a][b], ws[b], xs[a]);
        }
#pragma unroll
        for (; reads < (i + 1) * 4 * kWB / kProducts; ++reads) frag(u ^ 1, next, reads);
        if (u == 1) {
#pragma unroll
          for (; scales < (i + 1) * 2 * kWB / kProducts; ++scales) read_scale(t / 2 + 1, scales);
        }
#pragma unroll
        for (; loads < (i + 1) * kLoads / kProducts; ++loads) issue_one(t + u + kStages, slot, loads);
        __builtin_amdgcn_sched_barrier(0);
      }
      await_frags(u ^ 1);
      __builtin_amdgcn_sched_barrier(0);
      slot = next;
    }
    take_scales();
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tail's unused loads have left LDS alone

  // ---- epilogue: register e of acc[a][b]: token m0 + 32 kWB wi + 32 a + r, feature n0 + 32 kWB wj + 32 b +
  // 8 (e / 4) + 4 h + (e & 3)
  Out* out = (Out*)O.ptr + int64_t(slice) * M * N;
#pragma unroll
  for (int b = 0; b < kWB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int n = n0 + 32 * (kWB * wj + b) + 8 * g + 4 * h;
      float bv[4] = {0.f, 0.f, 0.f, 0.f};
      if (O.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) bv[e] = O.bias_f32 ? ((const float*)O.bias)[n + e] : bf16_to_f32(((const bf16_raw*)O.bias)[n + e]);
      }
#pragma unroll
      for (int a = 0; a < kWB; ++a) {
        const int m = m0 + 32 * (kWB * wi + a) + r;
        if (m >= M) continue;
        Out* dst = out + int64_t(m) * O.ld + n;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[a][b][4 * g + e] + bv[e];
        if (O.accumulate) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) v[e] += VecIO<Out>::load1(dst + e);
        }
        if (O.vec && n + 4 <= N) {
          if constexpr (sizeof(Out) == 2) {
            *reinterpret_cast<u32x2*>(dst) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
          } else {
            *reinterpret_cast<f32x4*>(dst) = f32x4{v[0], v[1], v[2], v[3]};
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) VecIO<Out>::store1(dst + e, v[e]);
        }
      }
    }
}

// out = (out +) bias + sum over slices, in slice order.
template <typename Out>
__global__ __launch_bounds__(kThreads) void fold_slices_kernel(const float* __restrict__ partial, int slices, int64_t total,
                                                               int N, const void* __restrict__ bias, bool bias_f32,
                                                               Out* __restrict__ out, bool accumulate) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= total) return;
  float v = 0.f;
  for (int s = 0; s < slices; ++s) v += partial[s * total + i];
  if (bias) {
    const int n = int(i % N);
    v += bias_f32 ? ((const float*)bias)[n] : bf16_to_f32(((const bf16_raw*)bias)[n]);
  }
  if (accumulate) v += VecIO<Out>::load1(out + i);
  VecIO<Out>::store1(out + i, v);
}

template <int kWB, typename Out, bool kWide>
void launch(const Operand& x, const Operand& w, const Output& o, int steps, int steps_per_slice, int slices,
            hipStream_t stream) {
  constexpr int kTile = 64 * kWB;
  constexpr int kLds = kStages * 2 * kTile * kStageK + 2 * 2 * kTile * 4;
  (void)hipFuncSetAttribute((const void*)fp8_gemm_kernel<kWB, Out, kWide>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  const int64_t tasks = ceil_div(x.rows, kTile) * ceil_div(w.rows, kTile) * slices;
  hipLaunchKernelGGL((fp8_gemm_kernel<kWB, Out, kWide>), dim3((unsigned)tasks), dim3(kThreads), kLds, stream, x, w, o, steps,
                     steps_per_slice);
}

}  // namespace

Fp8GemmPlan fp8_gemm_plan(int M, int N, int K, DType out_dtype) {
  Fp8GemmPlan p;
  const int steps = K / kStageK, groups = (steps + kGroupStages - 1) / kGroupStages;
  const int64_t big = ceil_div(M, 256) * ceil_div(N, 256);
  p.tile = big >= 192 && out_dtype == kBF16 ? 256 : 128;
  const int64_t tiles = ceil_div(M, p.tile) * ceil_div(N, p.tile);
  int slices = 1;
  const int slots = p.tile == 256 ? 256 : 512;  // workgroups the chip runs at once
  if (tiles < slots) slices = (int)(slots / tiles < groups ? slots / tiles : groups);
  if (slices < 1) slices = 1;
  const int per = (groups + slices - 1) / slices;
  p.steps_per_slice = per * kGroupStages;
  p.slices = (groups + per - 1) / per;
  return p;
}

void fp8_gemm(const Fp8Operand& x, const Fp8Operand& w, int K, const void* bias, DType bias_dtype, void* out,
              DType out_dtype, bool accumulate, const Fp8GemmPlan& plan, float* partial, hipStream_t stream) {
  const Operand X{(const uint8_t*)x.q, (const uint8_t*)x.scale, x.ld, x.ld_scale, x.rows, x.tiles ? 7 : 0};
  const Operand W{(const uint8_t*)w.q, (const uint8_t*)w.scale, w.ld, w.ld_scale, w.rows, w.tiles ? 7 : 0};
  const int N = w.rows, steps = K / kStageK;
  const bool split = plan.slices > 1;
  const DType kind = split ? kF32 : out_dtype;
  void* dst = split ? (void*)partial : out;
  const int quad = kind == kBF16 ? 8 : 16;
  const Output O{dst, split ? nullptr : bias, N, bias_dtype == kF32, !split && accumulate,
                 N % 4 == 0 && reinterpret_cast<uintptr_t>(dst) % quad == 0};
  auto go = [&](auto launcher) { launcher(X, W, O, steps, plan.steps_per_slice, plan.slices, stream); };
  if (out_dtype == kF32) go(launch<2, float, true>);
  else if (plan.tile == 256) kind == kBF16 ? go(launch<4, bf16_raw, false>) : go(launch<4, float, false>);
  else kind == kBF16 ? go(launch<2, bf16_raw, false>) : go(launch<2, float, false>);
  if (!split) return;
  const int64_t total = int64_t(x.rows) * N;
  const dim3 grid((unsigned)ceil_div(total, kThreads)), block(kThreads);
  if (out_dtype == kBF16)
    hipLaunchKernelGGL(fold_slices_kernel<bf16_raw>, grid, block, 0, stream, partial, plan.slices, total, N, bias,
                       bias_dtype == kF32, (bf16_raw*)out, accumulate);
  else
    hipLaunchKernelGGL(fold_slices_kernel<float>, grid, block, 0, stream, partial, plan.slices, total, N, bias,
                       bias_dtype == kF32, (float*)out, accumulate);
}

}  // namespace pda
