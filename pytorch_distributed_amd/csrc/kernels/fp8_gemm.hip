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
#include <type_traits>

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

struct Problem {
  Operand x, w;
  void* out;         // [M, N] (bf16 or fp32), or the fp32 partials [slices][M][N]
  const void* bias;  // [N] or null
  bool out_f32, bias_f32, vec;  // vec: rows are 16-byte aligned
  int steps, steps_per_slice, tasks;
};

// Up to two independent products in one launch (the two gradients of a layer): problem 1's workgroups follow
// problem 0's, padded to a multiple of 8 so that both see their XCD as blockIdx % 8.
struct Problems {
  Problem p[2];
};

template <int kWB, bool kWide>
__global__ __launch_bounds__(kThreads) void fp8_gemm_kernel(const Problems P) {
  constexpr int kTile = 64 * kWB;
  constexpr int kSlab = kTile * kStageK;       // bytes of one operand's stage
  constexpr int kStageBytes = 2 * kSlab;
  constexpr int kPieces = kTile / 64;          // 16-row loads per wave, stage and operand
  constexpr int kScaleLoads = kTile / 128;     // 64-row scale loads per wave and group (both operands)
  constexpr int kScaleBytes = 2 * kTile * 4;   // one group's scales: X rows, then W rows
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* scale_smem = smem + kStages * kStageBytes;
  float* bias_smem = reinterpret_cast<float*>(scale_smem + 2 * kScaleBytes);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave >> 1, wj = wave & 1;
  const int r = lane & 31, h = lane >> 5;

  const int padded0 = (P.p[0].tasks + 7) & ~7;
  const bool second = (int)blockIdx.x >= padded0;
  const Problem& pr = P.p[second];
  const int local = blockIdx.x - (second ? padded0 : 0);
  if (local >= pr.tasks) return;  // padding
  const Operand &X = pr.x, &W = pr.w;
  const int M = X.rows, N = W.rows;

  // Tasks are dealt to the 8 XCDs in contiguous ranges; consecutive tasks walk kGroupM token tiles x all
  // feature tiles, so the workgroups of an XCD share operand rows in its L2.
  const int tiles_m = (M + kTile - 1) / kTile, tiles_n = (N + kTile - 1) / kTile;
  const int n_tiles = tiles_m * tiles_n;
  const int q8 = pr.tasks / 8, r8 = pr.tasks % 8;
  const int xcd = local % 8, within = local / 8;
  const int task = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + within;
  const int slice = task / n_tiles;
  const int tile = task - slice * n_tiles;
  const int group = tile / (kGroupM * tiles_n);
  const int in_group = tile - group * (kGroupM * tiles_n);
  const int group_rows = min(kGroupM, tiles_m - group * kGroupM);
  const int m0 = (group * kGroupM + in_group % group_rows) * kTile;
  const int n0 = (in_group / group_rows) * kTile;
  const int first = slice * pr.steps_per_slice;  // a multiple of kGroupStages
  const int n_steps = min(pr.steps_per_slice, pr.steps - first);

  for (int i = threadIdx.x; i < kTile; i += kThreads) {  // read by the epilogue, many barriers from here
    float v = 0.f;
    if (pr.bias && n0 + i < N)
      v = pr.bias_f32 ? ((const float*)pr.bias)[n0 + i] : bf16_to_f32(((const bf16_raw*)pr.bias)[n0 + i]);
    bias_smem[i] = v;
  }

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
  __syncthreads();                                  // and nobody reads the ring any more: it stages the output

  // ---- epilogue: register e of acc[a][b]: token m0 + 32 kWB wi + 32 a + r, feature n0 + 32 kWB wj + 32 b +
  // 8 (e / 4) + 4 h + (e & 3). Through LDS, so that rows leave in whole lines: staged row = token, its 16-byte
  // chunks XOR-permuted with the token, so the lanes of a write (32 tokens, one feature offset) and of a read
  // (one token) both spread over the banks. Written in `passes` passes of the a-blocks that fit the ring.
  auto store_tile = [&](auto out_f32, auto passes) {
    using Out = std::conditional_t<decltype(out_f32)::value, float, bf16_raw>;
    constexpr int kRowBytes = kTile * (int)sizeof(Out), kVec = 16 / (int)sizeof(Out);
    constexpr int kPasses = decltype(passes)::value, kBlocks = kWB / kPasses, kRows = 64 * kBlocks;
    constexpr int kChunks = kRowBytes / 16;
    Out* out = (Out*)pr.out + int64_t(slice) * M * N;
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
#pragma unroll
      for (int ai = 0; ai < kBlocks; ++ai)
#pragma unroll
        for (int b = 0; b < kWB; ++b) {
          f32x16 v = acc[pass * kBlocks + ai][b];
          asm volatile("" : "+v"(v));  // one block at a time leaves the accumulator file
          const int row = 32 * (kBlocks * wi + ai) + r;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int col = 32 * (kWB * wj + b) + 8 * g + 4 * h;
            const f32x4 bv = *reinterpret_cast<const f32x4*>(bias_smem + col);
            const int at = row * kRowBytes + (((col / kVec) ^ (r & (kChunks - 1))) * 16) + (col % kVec) * (int)sizeof(Out);
            if constexpr (sizeof(Out) == 2)
              *reinterpret_cast<u32x2*>(smem + at) = u32x2{pack_bf16x2(v[4 * g] + bv[0], v[4 * g + 1] + bv[1]),
                                                          pack_bf16x2(v[4 * g + 2] + bv[2], v[4 * g + 3] + bv[3])};
            else
              *reinterpret_cast<f32x4*>(smem + at) = f32x4{v[4 * g] + bv[0], v[4 * g + 1] + bv[1], v[4 * g + 2] + bv[2], v[4 * g + 3] + bv[3]};
          }
        }
      __syncthreads();
      // staged row q is token 32 kWB (q / 32 / kBlocks) + 32 (pass kBlocks + q / 32 % kBlocks) + q % 32 of the tile
      auto token = [&](int q) {
        const int blk = q >> 5;
        return m0 + 32 * (kWB * (blk / kBlocks) + pass * kBlocks + blk % kBlocks) + (q & 31);
      };
      if (pr.vec) {
        const int ch = threadIdx.x % kChunks, n = n0 + ch * kVec;
        if (n < N) {  // (rows are whole chunks here)
#pragma unroll 4
          for (int q = threadIdx.x / kChunks; q < kRows; q += kThreads / kChunks) {
            const int m = token(q);
            const u32x4 w = *reinterpret_cast<const u32x4*>(smem + q * kRowBytes + ((ch ^ (q & 31 & (kChunks - 1))) * 16));
            if (m < M) *reinterpret_cast<u32x4*>(out + int64_t(m) * N + n) = w;
          }
        }
      } else {  // rows at any alignment: an element per lane, neighbours in neighbouring lanes
        const int col = threadIdx.x % kTile, n = n0 + col;
        if (n < N) {
#pragma unroll 4
          for (int q = threadIdx.x / kTile; q < kRows; q += kThreads / kTile) {
            const int m = token(q);
            const Out w = *reinterpret_cast<const Out*>(smem + q * kRowBytes + (((col / kVec) ^ (q & 31 & (kChunks - 1))) * 16) +
                                                        (col % kVec) * (int)sizeof(Out));
            if (m < M) out[int64_t(m) * N + n] = w;
          }
        }
      }
      if (pass + 1 < kPasses) __syncthreads();
    }
  };
  if constexpr (kWide) {
    store_tile(std::true_type{}, std::integral_constant<int, 1>{});
  } else if (pr.out_f32) {
    store_tile(std::true_type{}, std::integral_constant<int, kWB / 2>{});
  } else {
    store_tile(std::false_type{}, std::integral_constant<int, 1>{});
  }
}

// out = (out +) bias + sum over `slices` of partial [slices][total], in a fixed order. Up to three such sums in
// one launch. `tall`: many slices of few values (column sums): 64 values per workgroup, a quarter of the slices
// per wave; otherwise four values per thread.
struct Fold {
  const float* partial;
  const void* bias;
  void* out;
  int64_t total;
  int slices, N, blocks;
  bool bias_f32, out_f32, accumulate, tall;
};
struct Folds {
  Fold f[3];
};

__global__ __launch_bounds__(kThreads) void fold_kernel(const Folds folds) {
  __shared__ float red[4][64];
  int block = blockIdx.x, k = 0;
  while (block >= folds.f[k].blocks) block -= folds.f[k++].blocks;  // (the blocks' sum is the grid)
  const Fold& f = folds.f[k];
  auto finish = [&](int64_t i, float v) {
    if (f.bias) v += f.bias_f32 ? ((const float*)f.bias)[i % f.N] : bf16_to_f32(((const bf16_raw*)f.bias)[i % f.N]);
    if (f.out_f32) {
      float* o = (float*)f.out + i;
      *o = f.accumulate ? *o + v : v;
    } else {
      bf16_raw* o = (bf16_raw*)f.out + i;
      *o = f32_to_bf16(f.accumulate ? bf16_to_f32(*o) + v : v);
    }
  };
  if (f.tall) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = int64_t(block) * 64 + lane;
    float v = 0.f;
    if (i < f.total) {
#pragma unroll 8
      for (int s = wave; s < f.slices; s += 4) v += f.partial[s * f.total + i];
    }
    red[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && i < f.total) finish(i, (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
    return;
  }
  const int64_t i = (int64_t(block) * kThreads + threadIdx.x) * 4;
  if (f.total % 4 == 0) {
    if (i >= f.total) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < f.slices; ++s) {
      const f32x4 p = *reinterpret_cast<const f32x4*>(f.partial + s * f.total + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) finish(i + e, v[e]);
    return;
  }
  for (int e = 0; e < 4; ++e) {
    const int64_t at = int64_t(block) * kThreads * 4 + e * kThreads + threadIdx.x;
    if (at >= f.total) return;
    float v = 0.f;
#pragma unroll 4
    for (int s = 0; s < f.slices; ++s) v += f.partial[s * f.total + at];
    finish(at, v);
  }
}

template <int kWB, bool kWide>
void launch(const Problems& P, hipStream_t stream) {
  constexpr int kTile = 64 * kWB;
  constexpr int kLds = kStages * 2 * kTile * kStageK + 2 * 2 * kTile * 4 + kTile * 4;
  (void)hipFuncSetAttribute((const void*)fp8_gemm_kernel<kWB, kWide>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  const unsigned blocks = (unsigned)(((P.p[0].tasks + 7) & ~7) + P.p[1].tasks);
  hipLaunchKernelGGL((fp8_gemm_kernel<kWB, kWide>), dim3(blocks), dim3(kThreads), kLds, stream, P);
}

}  // namespace

// Which tile, and how many slices of the contraction: the smallest estimated time. The estimate is rounds of
// workgroups over the chip's slots, in microseconds fitted to measurements of 12 shapes from 16 x 3840 x 1280 to
// 8192 x 22016 x 4096 (most within 10 %). A stage of a 256 tile takes 0.72 with every compute unit busy (0.47
// alone); of a 128 tile 0.20 alone, 0.29 with one workgroup per compute unit, 0.60 with two. What else a
// workgroup costs (first loads, stores) is 10 and 3.3. So 8192 x 1280 x 5120 takes the 256 tile (160 of them: 65
// against 77), 2048^3 the 128 tile (13 against 28). A slice's partial sums are written and read again at some
// 4.5 TB/s and folded by a launch of 3: 1024 x 1024 x 8192 gains by four slices (33 -> 23), 2048^3 loses by two
// (13 -> 31). The widened products have the 128 tile only, at 1.5 times its stage.
static float plan_time(int tile, int64_t tasks, int steps, bool wide) {
  const int64_t slots = tile == 256 ? 256 : 512;
  auto round = [&](int64_t n) {
    const float load = n / 256.f;
    if (tile == 256) return 10.f + steps * (0.47f + 0.25f * load);
    const float stage = load <= 1.f ? 0.20f + 0.09f * load : 0.29f + 0.31f * (load - 1.f);
    return 3.3f + steps * stage * (wide ? 1.5f : 1.f);
  };
  const int64_t full = tasks / slots, rest = tasks % slots;
  return (tile == 256 ? 4.f : 1.4f) + full * round(slots) + (rest ? round(rest) : 0.f);
}

static Fp8GemmPlan plan_for_tile(int tile, int M, int N, int K, bool wide, float* time) {
  const int steps = K / kStageK, groups = (steps + kGroupStages - 1) / kGroupStages;
  const int64_t tiles = ceil_div(M, tile) * ceil_div(N, tile);
  Fp8GemmPlan best{tile, 1, groups * kGroupStages};
  *time = plan_time(tile, tiles, steps, wide);
  for (int slices = 2; slices <= groups && slices <= 16; ++slices) {
    const int per = (groups + slices - 1) / slices;
    const int real = (groups + per - 1) / per;  // slices that have any work
    if (real != slices) continue;
    const float t = plan_time(tile, tiles * slices, per * kGroupStages, wide) + 3.f + float(M) * N * (8.f * slices + 2.f) / 4.5e6f;
    if (t < *time) {
      *time = t;
      best = Fp8GemmPlan{tile, slices, per * kGroupStages};
    }
  }
  return best;
}

// Products that run together take the tile that is best for their sum, so that they share a launch.
void fp8_gemm_plan(Fp8GemmProblem* problems, int n) {
  Fp8GemmPlan plans[2][2];
  float sum[2] = {0.f, 0.f};
  bool wide = false;
  for (int i = 0; i < n; ++i) {
    Fp8GemmProblem& p = problems[i];
    wide |= p.out_dtype == kF32;
    for (int k = 0; k < 2; ++k) {
      float t;
      plans[k][i] = plan_for_tile(k ? 256 : 128, p.x.rows, p.w.rows, p.K, p.out_dtype == kF32, &t);
      sum[k] += t;
    }
  }
  const int k = !wide && sum[1] < sum[0];
  for (int i = 0; i < n; ++i) problems[i].plan = plans[k][i];
}

void fp8_gemm(const Fp8GemmProblem* problems, int n, const Fp8ColumnSums* sums, hipStream_t stream) {
  Problem ps[2] = {};
  Folds folds = {};
  int n_folds = 0;
  auto add_fold = [&](Fold f) {
    f.blocks = (int)(f.tall ? ceil_div(f.total, 64) : ceil_div(f.total, kThreads * 4));
    folds.f[n_folds++] = f;
  };
  for (int i = 0; i < n; ++i) {
    const Fp8GemmProblem& g = problems[i];
    auto operand = [](const Fp8Operand& o) {
      return Operand{(const uint8_t*)o.q, (const uint8_t*)o.scale, o.ld, o.ld_scale, o.rows, o.tiles ? 7 : 0};
    };
    const int M = g.x.rows, N = g.w.rows;
    const bool fold = g.partial != nullptr;
    const bool f32 = fold || g.out_dtype == kF32;
    void* out = fold ? (void*)g.partial : g.out;
    const int64_t tasks = ceil_div(M, g.plan.tile) * ceil_div(N, g.plan.tile) * g.plan.slices;
    ps[i] = Problem{operand(g.x), operand(g.w), out, fold ? nullptr : g.bias, f32, g.bias_dtype == kF32,
                    (int64_t(N) * (f32 ? 4 : 2)) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                    g.K / kStageK, g.plan.steps_per_slice, (int)tasks};
    if (fold)
      add_fold(Fold{g.partial, g.bias, g.out, int64_t(M) * N, g.plan.slices, N, 0, g.bias_dtype == kF32, g.out_dtype == kF32,
                    g.accumulate, false});
  }
  auto go = [&](const Problem& a, const Problem* b, int tile, bool wide) {
    Problems P = {{a, b ? *b : Problem{}}};
    if (wide) launch<2, true>(P, stream);
    else if (tile == 256) launch<4, false>(P, stream);
    else launch<2, false>(P, stream);
  };
  auto wide = [&](int i) { return problems[i].out_dtype == kF32; };
  if (n == 2 && problems[0].plan.tile == problems[1].plan.tile && wide(0) == wide(1)) {
    const int longer = ps[1].steps_per_slice > ps[0].steps_per_slice;  // long tasks first: the short ones fill up
    go(ps[longer], &ps[1 - longer], problems[0].plan.tile, wide(0));
  } else {
    for (int i = 0; i < n; ++i) go(ps[i], nullptr, problems[i].plan.tile, wide(i));
  }
  if (sums)
    add_fold(Fold{sums->partial, nullptr, sums->out, sums->C, sums->blocks, sums->C, 0, false, sums->out_dtype == kF32,
                  sums->accumulate, true});
  if (n_folds == 0) return;
  unsigned blocks = 0;
  for (int i = 0; i < n_folds; ++i) blocks += (unsigned)folds.f[i].blocks;
  hipLaunchKernelGGL(fold_kernel, dim3(blocks), dim3(kThreads), 0, stream, folds);
}

}  // namespace pda
