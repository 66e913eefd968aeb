// Block-scaled 8-bit matrix product for gfx950:
//   out[M, N] = (bias[N] +) sum_k 2^(ex[m, k/128] + ew[n, k/128]) x[m, k] w[n, k],   x, w e4m3, fp32 accumulation.
//
// Both operands are contraction-contiguous, rows padded with zeros to a multiple of 128 values; the
// scales are bytes e + 127, one per 128 values of a row or per 128 x 128 tile. v_mfma_scale_f32_32x32x64
// takes such a byte per row and applies it inside the instruction, so a block-scaled product costs no
// vector instruction per product more than an unscaled one.
//
// Structure. A workgroup of 4 waves (2 x 2) owns an output tile of 128 x 128, 256 x 192 or 256 x 256 (tokens x
// features), each wave a quarter as kA x kB blocks of 32 x 32. A pipeline stage is 64 values of the contraction:
// [tile rows][64 bytes] of each operand, moved global -> LDS by buffer loads into a ring of four. The body of stage t
//   * waits until stage t + 1 has landed (counted: two younger stages stay in flight) and meets the
//     other waves, who by then have read stage t out of LDS;
//   * issues the products of stage t from registers, and between them the LDS reads of stage t + 1 and
//     the loads of stage t + 4 into the slot that stage t has left.
// One barrier per 16 matrix instructions (1,024 matrix cycles) of a wave at 256 x 256.
// Large tiles (one workgroup per compute unit): a workgroup takes several tiles, and the stages run on across
// them: while a tile is rounded and stored, the next one's first four stages are on their way. Measured against
// a workgroup per tile: 8192 x 5120 x 1280 (640 tiles) 84 -> 72 us, 8192 x 22016 x 4096 (2,752) 665 -> 591.
// What bounds it: the matrix pipes at the clock that the power leaves. 8192 x 22016 x 4096 runs at 2,500 TFLOP/s
// (a library product of 8192^3 at 2,593); short contractions pay some 3 us a tile for the epilogue.
// 128 tile: two workgroups per compute unit cover each other's first loads and epilogue.
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
// instead: fragments widened to bf16 on the way to v_mfma_f32_32x32x16_bf16, scale included (exact: see widen2), whose
// sums are good to 6e-8, at half the matrix rate (1003 x 1601 x 777: 12.1 us).
//
// Few output tiles (weight gradients, few tokens): the contraction is cut into slices of whole 512-value
// scale groups, fp32 partial tiles are folded in slice order by a second kernel (deterministic).
#include <algorithm>
#include <type_traits>

#include "attention_common.h"
#include "pda_kernels.h"

namespace pda {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef u32x4 __attribute__((aligned(2))) u32x4_anywhere;  // 16 bytes of global memory at any alignment

constexpr int kThreads = 256;
constexpr int kStages = 4;
constexpr int kStageK = 64;                 // values (bytes) of the contraction per stage
constexpr int kGroupStages = 8;             // stages whose scales are fetched together: 4 blocks of 128, a dword a row
constexpr int kSlots = 256;                 // workgroups of the 256 tile at once: one per compute unit
constexpr int kGroupM = 4;                  // token tiles walked together by consecutive tasks

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

// Two of the e4m3 values of `v` (its lower or upper half) times 2^(byte - 127) as bf16: exact for bytes of 3 and more
// (e4m3 has 4 significant bits and its smallest number is 2^-9; bf16's is 2^-133, and the matrix instruction takes
// subnormal operands). At bytes 0 to 2, blocks whose largest magnitude is at most 448 * 2^-125, it rounds to multiples of
// 2^-133.
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
  bool out_f32, bias_f32;
  int steps, steps_per_slice, tasks;
};

// Up to two independent products in one launch (the two gradients of a layer): problem 1's tasks follow problem 0's.
struct Problems {
  Problem p[2];
};

// The output tile and the slice of the contraction of one task.
struct Place {
  int which, slice, m0, n0, first, n_steps;  // which < 0: none
};

// Task `round` of workgroup `w` of `grid`: a round is the next `grid` tasks, every other one is dealt backwards
// (whoever had a long task then gets a short one). Within a round, and within a problem, the 8 XCDs get contiguous
// ranges; consecutive tasks walk kGroupM token tiles x all feature tiles, so an XCD's workgroups share operand
// rows in its L2.
template <int kTileM, int kTileN>
__device__ __forceinline__ Place place_of(const Problems& P, int w, int grid, int round) {
  const int base = round * grid, left = P.p[0].tasks + P.p[1].tasks - base;
  const int count = min(grid, left);
  if (round & 1) w = grid - 1 - w;
  Place at;
  at.which = -1;
  if (w >= count) return at;
  const int c0 = max(min(P.p[0].tasks - base, count), 0);
  const bool second = w >= c0;
  const int n = second ? count - c0 : c0, j = second ? w - c0 : w;
  const int q8 = n / 8, r8 = n % 8, x = j % 8;
  const int task = base + (second ? c0 - P.p[0].tasks : 0) + (x < r8 ? x * (q8 + 1) : r8 * (q8 + 1) + (x - r8) * q8) + j / 8;
  const Problem& pr = P.p[second];
  const int tiles_m = (pr.x.rows + kTileM - 1) / kTileM, tiles_n = (pr.w.rows + kTileN - 1) / kTileN;
  const int n_tiles = tiles_m * tiles_n;
  const int slice = task / n_tiles;
  const int tile = task - slice * n_tiles;
  const int group = tile / (kGroupM * tiles_n);
  const int in_group = tile - group * (kGroupM * tiles_n);
  const int group_rows = min(kGroupM, tiles_m - group * kGroupM);
  at.which = second;
  at.slice = slice;
  at.m0 = (group * kGroupM + in_group % group_rows) * kTileM;
  at.n0 = (in_group / group_rows) * kTileN;
  at.first = slice * pr.steps_per_slice;  // a multiple of kGroupStages
  at.n_steps = min(pr.steps_per_slice, pr.steps - at.first);
  return at;
}

constexpr int kScaleRing = 4;  // scale groups in LDS: loads run at most 4 stages ahead, at least 2 stages (one group) a tile
constexpr int kBiasRing = 4;   // likewise of tiles

// kA x kB: blocks of 32 tokens x 32 features of a wave; four waves (2 x 2) to a tile.
constexpr bool streams(int kA) { return kA == 4; }  // several tiles per workgroup, as one stream of stages
constexpr int wave_turn_bytes(int kB) { return 32 * (kB == 3 ? 192 : 128); }  // LDS a wave turns 32 tokens of its output around in
constexpr int lds_bytes(int kA, int kB) {
  const int m = 64 * kA, n = 64 * kB;
  const int ring = kStages * (m + n) * kStageK, scales = kScaleRing * 2 * m * 4;
  return streams(kA) ? ring + scales + kBiasRing * n * 4 + 4 * wave_turn_bytes(kB) : ring + scales + n * 4;
}

// Wait until at most so many vector memory operations of this wave are left.
template <int kLeft>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kLeft) : "memory");
}

template <int kA, int kB, bool kWide>
__global__ __launch_bounds__(kThreads) void fp8_gemm_kernel(const Problems P) {
  constexpr bool kStream = streams(kA);
  constexpr int kTileM = 64 * kA, kTileN = 64 * kB;
  constexpr int kSlab = kTileM * kStageK;      // bytes of X's part of a stage
  constexpr int kStageBytes = (kTileM + kTileN) * kStageK;
  constexpr int kLoads = kA + kB;              // 16-row loads per wave and stage: kA of X, then kB of W
  constexpr int kScaleLoads = kTileM / 128;    // 64-row scale loads per wave and group (both operands)
  constexpr int kScaleBytes = 2 * kTileM * 4;  // one group's scales: X rows, then W rows
  constexpr int kStores = kB == 3 ? 24 : 32;   // of a wave in an epilogue, at least
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* scale_smem = smem + kStages * kStageBytes;
  char* bias_smem = scale_smem + kScaleRing * kScaleBytes;
  [[maybe_unused]] char* turn_smem = bias_smem + kBiasRing * kTileN * 4;  // (kStream)

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave >> 1, wj = wave & 1;
  const int r = lane & 31, h = lane >> 5;

  Place at = place_of<kTileM, kTileN>(P, blockIdx.x, gridDim.x, 0);  // what is computed; every workgroup has a first task
  if constexpr (!kStream) {
    const Problem& pr = P.p[at.which];
    for (int i = threadIdx.x; i < kTileN; i += kThreads) {  // read by the epilogue, many barriers from here
      float v = 0.f;
      if (pr.bias && at.n0 + i < pr.w.rows)
        v = pr.bias_f32 ? ((const float*)pr.bias)[at.n0 + i] : bf16_to_f32(((const bf16_raw*)pr.bias)[at.n0 + i]);
      reinterpret_cast<float*>(bias_smem)[i] = v;
    }
  }

  // ---- staging: the loads' own cursor, kStages stages ahead of the products and across tiles.
  // Piece i of a slab = rows (rows / 4) wave + 16 i .. +15, lane p -> row + p / 4, slot p % 4.
  // Rows past the end repeat the last one (never stored).
  // (All offsets fit 32 bits: a tile's rows span at most 256 * 2^22 bytes, a bound the host checks.)
  // Scales: group g = blocks 4 g .. 4 g + 3 of the slice, a dword per row; 64 rows per load, all of one operand:
  // waves 0, 1 fetch the scales of X's rows, waves 2, 3 those of W's.
  __amdgpu_buffer_rsrc_t x_src, w_src, s_src;
  unsigned off[kLoads], s_off[kScaleLoads];
  int c_round = 0, c_step = 0, c_steps = 0, c_groups = 0;
  bool c_done = false;
  auto aim = [&](const Place& to) {
    const Operand &X = P.p[to.which].x, &W = P.p[to.which].w;
    const int x_rows = min(X.rows - to.m0, kTileM), w_rows = min(W.rows - to.n0, kTileN);
    const unsigned k_bytes = (unsigned)to.n_steps * kStageK;
    x_src = bounded(X.q + int64_t(to.m0) * X.ld + int64_t(to.first) * kStageK, (unsigned)(x_rows - 1) * (unsigned)X.ld + k_bytes);
    w_src = bounded(W.q + int64_t(to.n0) * W.ld + int64_t(to.first) * kStageK, (unsigned)(w_rows - 1) * (unsigned)W.ld + k_bytes);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool of_x = i < kA;
      const int row = of_x ? 16 * kA * wave + 16 * i + (lane >> 2) : 16 * kB * wave + 16 * (i - kA) + (lane >> 2);
      const unsigned chunk = (unsigned)(((lane & 3) ^ ((row >> 2) & 3)) * 16);
      off[i] = (unsigned)min(row, (of_x ? x_rows : w_rows) - 1) * (unsigned)(of_x ? X.ld : W.ld) + chunk;
    }
    const Operand& s_op = wave < 2 ? X : W;
    const int s_row0 = wave < 2 ? to.m0 : to.n0, s_last = s_op.rows - 1;
    const int s_lo = s_row0 >> s_op.shift, s_hi = min(s_row0 + kTileM - 1, s_last) >> s_op.shift;
    s_src = bounded(s_op.scale + int64_t(s_lo) * s_op.ld_scale + to.first / 2,
                    (unsigned)(s_hi - s_lo) * (unsigned)s_op.ld_scale + 4u * (unsigned)((to.n_steps + kGroupStages - 1) / kGroupStages));
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
      const int row = ((wave & 1) * kScaleLoads + i) * 64 + lane;
      s_off[i] = (unsigned)((min(s_row0 + row, s_last) >> s_op.shift) - s_lo) * (unsigned)s_op.ld_scale;
    }
    c_step = 0;
    c_steps = to.n_steps;
    if constexpr (kStream) {
      // the tile's bias as it lies there, fp32 or pairs of bf16 (whole dwords: 4-byte aligned, a bound the host checks)
      const Problem& pr = P.p[to.which];
      if (pr.bias && wave * 256 < kTileN * (pr.bias_f32 ? 4 : 2)) {
        const unsigned size = pr.bias_f32 ? 4u : 2u;
        const auto b_src = bounded((const uint8_t*)pr.bias + (unsigned)to.n0 * size, ((unsigned)w_rows * size + 3u) & ~3u);
        load_to_lds4(b_src, (unsigned)(wave * 64 + lane) * 4u, 0, bias_smem + (c_round & (kBiasRing - 1)) * kTileN * 4 + wave * 256);
      }
    }
  };
  // Before the loads of an even stage: on to the next tile where this one ends (after the last, its last two stages
  // again, never used), and the scales of a new group.
  auto turn = [&]() {
    if (c_step == c_steps) {
      Place to;
      to.which = -1;
      if constexpr (kStream) {
        if (!c_done) to = place_of<kTileM, kTileN>(P, blockIdx.x, gridDim.x, ++c_round);
      }
      if (to.which < 0) {
        c_done = true;
        c_step = c_steps - 2;
      } else {
        aim(to);
      }
    }
    if ((c_step & (kGroupStages - 1)) == 0 && !c_done) {
#pragma unroll
      for (int i = 0; i < kScaleLoads; ++i)
        load_to_lds4(s_src, s_off[i], 4u * (unsigned)(c_step / kGroupStages),
                     scale_smem + (c_groups & (kScaleRing - 1)) * kScaleBytes + (wave * kScaleLoads + i) * 256);
      ++c_groups;
    }
  };
  auto issue_one = [&](int slot, int i) {  // i < kLoads
    const unsigned ko = (unsigned)c_step * kStageK;
    char* dst = smem + slot * kStageBytes;
    if (i < kA) load_to_lds16(x_src, off[i], ko, dst + (16 * kA * wave + 16 * i) * kStageK);
    else load_to_lds16(w_src, off[i], ko, dst + kSlab + (16 * kB * wave + 16 * (i - kA)) * kStageK);
  };

  f32x16 acc[kA][kB];

  // ---- fragment addresses: lane (r, h) reads chunks h and 2 + h of row r of each 32-row block
  const unsigned smem_base = lds_addr(smem);
  const int f = (r >> 2) & 3;
  const unsigned c0 = (unsigned)((h ^ f) << 4), c1 = (unsigned)(((2 + h) ^ f) << 4);
  const unsigned x_row = (unsigned)((32 * kA * wi + r) * kStageK);
  const unsigned w_row = (unsigned)(kSlab + (32 * kB * wj + r) * kStageK);
  u32x4 xf[2][kA][2], wf[2][kB][2];
  constexpr int kReads = 2 * (kA + kB);
  // read i of the fragments of the stage in `slot`: w0 x0 w1 x1 ..., two chunks each, what x has more at the end
  auto frag = [&](int buf, int slot, int i) {
    const unsigned base = smem_base + slot * kStageBytes;
    const bool of_x = i >= 4 * kB || (i & 2);
    const int blk = i >= 4 * kB ? kB + (i - 4 * kB) / 2 : i >> 2;
    const unsigned at = base + (of_x ? x_row : w_row) + ((i & 1) ? c1 : c0);
    u32x4& dst = of_x ? xf[buf][blk][i & 1] : wf[buf][blk][i & 1];
    if (blk == 0) dst = chunk_read<0>(at);
    if (blk == 1) dst = chunk_read<2048>(at);
    if (blk == 2) dst = chunk_read<4096>(at);
    if (blk == 3) dst = chunk_read<6144>(at);
  };
  // the values read by `frag` exist after this point (ties every register to the wait)
  auto await_frags = [&](int buf) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int a = 0; a < kA; ++a) asm volatile("" : "+v"(xf[buf][a][0]), "+v"(xf[buf][a][1]));
#pragma unroll
    for (int b = 0; b < kB; ++b) asm volatile("" : "+v"(wf[buf][b][0]), "+v"(wf[buf][b][1]));
  };
  // scale bytes of the next block (a pair of stages), read i: X's 32-row blocks, then W's
  const unsigned scale_base = lds_addr(scale_smem);
  const unsigned xs_row = (unsigned)((32 * kA * wi + r) * 4), ws_row = (unsigned)((kTileM + 32 * kB * wj + r) * 4);
  uint32_t xs[kA], ws[kB], xs_next[kA], ws_next[kB];
  unsigned scale_at = scale_base;  // of the block that is read next
  int block = 0, groups = 0;       // its place: block of the tile, group of the workgroup's stream
  auto next_block = [&](bool tile_ends) {
    block = tile_ends ? 0 : block + 1;
    if ((block & 3) == 0) ++groups;
    scale_at = scale_base + (groups & (kScaleRing - 1)) * kScaleBytes + (block & 3);
  };
  auto read_scale = [&](int i) {
    const bool of_x = i < kA;
    const unsigned at = scale_at + (of_x ? xs_row : ws_row);
    const int blk = of_x ? i : i - kA;
    uint32_t& dst = of_x ? xs_next[blk] : ws_next[blk];
    if (blk == 0) asm volatile("ds_read_u8 %0, %1" : "=v"(dst) : "v"(at));
    if (blk == 1) asm volatile("ds_read_u8 %0, %1 offset:128" : "=v"(dst) : "v"(at));
    if (blk == 2) asm volatile("ds_read_u8 %0, %1 offset:256" : "=v"(dst) : "v"(at));
    if (blk == 3) asm volatile("ds_read_u8 %0, %1 offset:384" : "=v"(dst) : "v"(at));
  };
  auto take_scales = [&]() {  // after await_frags
#pragma unroll
    for (int a = 0; a < kA; ++a) {
      asm volatile("" : "+v"(xs_next[a]));
      xs[a] = xs_next[a];
    }
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      asm volatile("" : "+v"(ws_next[b]));
      ws[b] = ws_next[b];
    }
  };

  aim(at);
#pragma unroll
  for (int t = 0; t < kStages; ++t) {
    if (t % 2 == 0) turn();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) issue_one(t, i);
    ++c_step;
  }
  wait_vm<3 * kLoads>();
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < kA + kB; ++i) read_scale(i);
#pragma unroll
  for (int i = 0; i < kReads; ++i) frag(0, 0, i);
  await_frags(0);
  take_scales();

  int slot = 0;   // of the stage in hand
  int fresh = 0;  // stages since an epilogue left its stores in flight: see below
  for (int round = 0;;) {
#pragma unroll
    for (int a = 0; a < kA; ++a)
#pragma unroll
      for (int b = 0; b < kB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;

    for (int t = 0; t < at.n_steps; t += 2) {  // n_steps is even; a pair of stages is one scale block
      next_block(t + 2 == at.n_steps);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // Stage t + u + 1 has landed: two younger stages may be in flight (anything else among them makes the count
        // strict by that much), and in the first three stages after an epilogue its stores too, which lie between
        // that stage and the youngest. After the barrier everyone's part has, and nobody reads this slot any more.
        if constexpr (kStream) {
          // (the branch is inside the block: around a branch of its own the compiler would sink products)
          asm volatile("s_cmp_gt_i32 %0, 0\n\ts_cbranch_scc1 .Lfresh%=\n\ts_waitcnt vmcnt(%1)\n.Lfresh%=:\n\ts_waitcnt vmcnt(%2)"
                       ::"s"(__builtin_amdgcn_readfirstlane(fresh)), "i"(2 * kLoads), "i"(2 * kLoads + kStores)
                       : "memory", "scc");
          fresh = max(fresh - 1, 0);
        } else {
          wait_vm<2 * kLoads>();
        }
        __builtin_amdgcn_s_barrier();
        if (u == 0) turn();
        __builtin_amdgcn_sched_barrier(0);
        const int next = (slot + 1) & (kStages - 1);
        constexpr int kProducts = kA * kB;
        int reads = 0, loads = 0, scales = 0;
        [[maybe_unused]] bf16x8 xb[4], wb[kWide ? kB : 1][4];
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
          const int a = i / kB, b = i % kB;
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
          for (; reads < (i + 1) * kReads / kProducts; ++reads) frag(u ^ 1, next, reads);
          if (u == 1) {
#pragma unroll
            for (; scales < (i + 1) * (kA + kB) / kProducts; ++scales) read_scale(scales);
          }
#pragma unroll
          for (; loads < (i + 1) * kLoads / kProducts; ++loads) issue_one(slot, loads);
          __builtin_amdgcn_sched_barrier(0);
        }
        ++c_step;
        await_frags(u ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        slot = next;
      }
      take_scales();
    }

    // ---- epilogue: register e of acc[a][b]: token m0 + 32 kA wi + 32 a + r, feature n0 + 32 kB wj + 32 b +
    // 8 (e / 4) + 4 h + (e & 3). Through LDS, so that rows leave in whole lines: staged row = token, its 16-byte
    // chunks XOR-permuted with the token, so the lanes of a write (32 tokens, one feature offset) and of a read
    // (whole tokens) both spread over the banks.
    const Problem& pr = P.p[at.which];
    const int M = pr.x.rows, N = pr.w.rows;
    const int m0 = at.m0, n0 = at.n0;
    const int64_t slice0 = int64_t(at.slice) * M * N;
    if constexpr (kStream) {
      // The next tile's loads are on their way and its first fragments in registers: a wave turns its quarter around
      // in LDS of its own, 32 tokens x 128 (kB = 3: 192) bytes at a time, meets nobody, and goes on without waiting for its
      // stores. LDS by inline assembly (in order within a wave): the compiler would wait for the loads in flight.
#pragma unroll
      for (int a = 0; a < kA; ++a)
#pragma unroll
        for (int b = 0; b < kB; ++b) asm volatile("" : "+a"(acc[a][b]));
      int el = lane;
      asm volatile("" : "+v"(el));  // (addresses are formed here, not held through the products)
      const int er = el & 31, eh = el >> 5;
      const int bias_f32 = __builtin_amdgcn_readfirstlane(pr.bias_f32);
      const int has_bias = __builtin_amdgcn_readfirstlane(pr.bias != nullptr);  // (held: not fetched after every store)
      auto store_quarter = [&](auto out_f32) {
        using Out = std::conditional_t<decltype(out_f32)::value, float, bf16_raw>;
        constexpr int kSize = (int)sizeof(Out), kVec = 16 / kSize;
        constexpr int kT = kSize == 4 ? 1 : kB == 3 ? 3 : 2;                  // feature blocks turned together
        constexpr int kRow = 32 * kT * kSize, kChunks = kRow / 16;            // bytes and chunks of a token
        constexpr int kMoves = 32 * kChunks / 64, kSwap = kChunks == 8 ? 7 : 3;  // chunks XORed with the token's low bits
        Out* out = (Out*)pr.out + slice0 + int64_t(m0) * N;
        const auto dst = __builtin_amdgcn_make_buffer_rsrc((void*)out, 0, (int)((unsigned)min(M - m0, kTileM) * (unsigned)N * kSize), 0x00027000);
        const unsigned turn_base = lds_addr(turn_smem) + wave * wave_turn_bytes(kB);
        const unsigned bias_base = lds_addr(bias_smem) + (round & (kBiasRing - 1)) * kTileN * 4;
#pragma unroll
        for (int b0 = 0; b0 < kB; b0 += kT) {
          f32x4 bv[kT][4];
#pragma unroll
          for (int i = 0; i < 4 * kT; ++i) bv[i / 4][i % 4] = f32x4{0.f, 0.f, 0.f, 0.f};
          const unsigned b_col = (unsigned)(32 * (kB * wj + b0) + 4 * eh);
          if (has_bias && bias_f32) {
#pragma unroll
            for (int i = 0; i < 4 * kT; ++i) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(bv[i / 4][i % 4]) : "v"(bias_base + b_col * 4), "i"(32 * i));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < 4 * kT; ++i) asm volatile("" : "+v"(bv[i / 4][i % 4]));
          } else if (has_bias) {
            u32x2 w[4 * kT];
#pragma unroll
            for (int i = 0; i < 4 * kT; ++i) asm volatile("ds_read_b64 %0, %1 offset:%2" : "=v"(w[i]) : "v"(bias_base + b_col * 2), "i"(16 * i));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < 4 * kT; ++i) {
              asm volatile("" : "+v"(w[i]));
              bv[i / 4][i % 4] = f32x4{__uint_as_float(w[i][0] << 16), __uint_as_float(w[i][0] & 0xffff0000u),
                                       __uint_as_float(w[i][1] << 16), __uint_as_float(w[i][1] & 0xffff0000u)};
            }
          }
          // lane l moves chunk (64 i + l) % kChunks of token (64 i + l) / kChunks
          unsigned from[kMoves], to_at[kMoves];
          int to_col[kMoves];
#pragma unroll
          for (int i = 0; i < kMoves; ++i) {
            const int token = (64 * i + el) / kChunks, chunk = (64 * i + el) % kChunks;
            from[i] = turn_base + token * kRow + ((chunk ^ (token & kSwap)) << 4);
            to_col[i] = n0 + 32 * (kB * wj + b0) + chunk * kVec;
            to_at[i] = ((unsigned)(32 * kA * wi + token) * (unsigned)N + (unsigned)to_col[i]) * kSize;
          }
          const bool ragged = N % kVec != 0 && n0 + 32 * (kB * wj + b0 + kT) > N;
          using Piece = std::conditional_t<kSize == 2, u32x2, f32x4>;  // four features of a token
          Piece piece[kT][4];
          auto round_up = [&](int a) {  // one block at a time leaves the accumulator file
#pragma unroll
            for (int b = 0; b < kT; ++b) {
              f32x16 v = acc[a][b0 + b];
              asm volatile("" : "+v"(v));
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const f32x4 y = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]} + bv[b][g];
                if constexpr (kSize == 2) piece[b][g] = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
                else piece[b][g] = y;
              }
            }
          };
          round_up(0);
#pragma unroll
          for (int a = 0; a < kA; ++a) {
#pragma unroll
            for (int b = 0; b < kT; ++b)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const unsigned chunk = (unsigned)(32 * b + 8 * g + 4 * eh) / kVec;
                const unsigned to = turn_base + er * kRow + ((chunk ^ (er & kSwap)) << 4) + (kSize == 2 ? 8 * eh : 0);
                if constexpr (kSize == 2) asm volatile("ds_write_b64 %0, %1" ::"v"(to), "v"(piece[b][g]) : "memory");
                else asm volatile("ds_write_b128 %0, %1" ::"v"(to), "v"(piece[b][g]) : "memory");
              }
            u32x4 w[kMoves];
#pragma unroll
            for (int i = 0; i < kMoves; ++i) w[i] = chunk_read<0>(from[i]);
            if (a + 1 < kA) round_up(a + 1);  // while they come
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < kMoves; ++i) asm volatile("" : "+v"(w[i]));
            // Rows at any alignment. Out of range (rows past M, pieces past or across N): dropped, but issued and counted.
            const unsigned down = (unsigned)(32 * a * N) * kSize;
#pragma unroll
            for (int i = 0; i < kMoves; ++i)
              __builtin_amdgcn_raw_buffer_store_b128(w[i], dst, (int)(to_col[i] + kVec <= N ? to_at[i] + down : 0x80000000u), 0, 0);
            if (ragged) {  // wave-uniform: the piece across N, one element at a time
#pragma unroll
              for (int i = 0; i < kMoves; ++i)
#pragma unroll
                for (int e = 0; e + 1 < kVec; ++e) {
                  const unsigned to = to_col[i] + kVec > N && to_col[i] + e < N ? to_at[i] + down + e * kSize : 0x80000000u;
                  if constexpr (kSize == 4) __builtin_amdgcn_raw_buffer_store_b32(w[i][e], dst, (int)to, 0, 0);
                  else __builtin_amdgcn_raw_buffer_store_b16((unsigned short)(w[i][e / 2] >> (16 * (e & 1))), dst, (int)to, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      };
      // (at least kStores stores of a wave: the count of the three stages that follow)
      if (pr.out_f32) store_quarter(std::true_type{});
      else store_quarter(std::false_type{});
      fresh = 3;
      at = place_of<kTileM, kTileN>(P, blockIdx.x, gridDim.x, ++round);
      if (at.which < 0) break;
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tail's unused loads have left LDS alone
      __syncthreads();                                  // and nobody reads the ring any more: it stages the output
      auto store_tile = [&](auto out_f32) {
        using Out = std::conditional_t<decltype(out_f32)::value, float, bf16_raw>;
        constexpr int kRowBytes = kTileN * (int)sizeof(Out), kVec = 16 / (int)sizeof(Out);
        constexpr int kChunks = kRowBytes / 16;
        Out* out = (Out*)pr.out + slice0;
#pragma unroll
        for (int a = 0; a < kA; ++a)
#pragma unroll
          for (int b = 0; b < kB; ++b) {
            f32x16 v = acc[a][b];
            asm volatile("" : "+v"(v));  // one block at a time leaves the accumulator file
            const int row = 32 * (kA * wi + a) + r;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int col = 32 * (kB * wj + b) + 8 * g + 4 * h;
              const f32x4 bv = *reinterpret_cast<const f32x4*>(bias_smem + col * 4);
              const int to = row * kRowBytes + (((col / kVec) ^ (r & (kChunks - 1))) * 16) + (col % kVec) * (int)sizeof(Out);
              if constexpr (sizeof(Out) == 2)
                *reinterpret_cast<u32x2*>(smem + to) = u32x2{pack_bf16x2(v[4 * g] + bv[0], v[4 * g + 1] + bv[1]),
                                                            pack_bf16x2(v[4 * g + 2] + bv[2], v[4 * g + 3] + bv[3])};
              else
                *reinterpret_cast<f32x4*>(smem + to) = f32x4{v[4 * g] + bv[0], v[4 * g + 1] + bv[1], v[4 * g + 2] + bv[2], v[4 * g + 3] + bv[3]};
            }
          }
        __syncthreads();
        const int ch = threadIdx.x % kChunks, n = n0 + ch * kVec;
        if (n < N) {
#pragma unroll 4
          for (int q = threadIdx.x / kChunks; q < kTileM; q += kThreads / kChunks) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(smem + q * kRowBytes + ((ch ^ (q & 31 & (kChunks - 1))) * 16));
            if (m0 + q >= M) break;
            Out* to = out + int64_t(m0 + q) * N + n;
            if (n + kVec <= N) {
              *reinterpret_cast<u32x4_anywhere*>(to) = w;
            } else {
#pragma unroll
              for (int e = 0; e + 1 < kVec; ++e)
                if (n + e < N) {
                  if constexpr (sizeof(Out) == 4) to[e] = __uint_as_float(w[e]);
                  else to[e] = (bf16_raw)(w[e / 2] >> (16 * (e & 1)));
                }
            }
          }
        }
      };
      if (kWide || pr.out_f32) store_tile(std::true_type{});
      else if constexpr (!kWide) store_tile(std::false_type{});
      break;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (kStream) no load to LDS outlives the workgroup
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

template <int kA, int kB, bool kWide>
void launch(const Problems& P, hipStream_t stream) {
  constexpr int kLds = lds_bytes(kA, kB);
  (void)hipFuncSetAttribute((const void*)fp8_gemm_kernel<kA, kB, kWide>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  const int tasks = P.p[0].tasks + P.p[1].tasks;
  const unsigned blocks = (unsigned)(streams(kA) ? std::min(tasks, kSlots) : tasks);
  hipLaunchKernelGGL((fp8_gemm_kernel<kA, kB, kWide>), dim3(blocks), dim3(kThreads), kLds, stream, P);
}

}  // namespace

// Which tile, and how many slices of the contraction: the smallest estimated time, in microseconds fitted to
// measurements of 14 shapes from 16 x 3840 x 1280 to 8192 x 22016 x 4096 (most within 10 %).
// 256 tile: workgroups stream through their tasks, dealt as place_of does; a stage takes 0.75 with every compute
// unit busy (0.47 alone), a tile 3 more (its epilogue), the launch 10 (first loads, last stores). The 192 tile takes
// 0.61 (0.37) a stage: dearer per product, but it fills a round that 256 leaves half empty.
// 128 tile: rounds of workgroups over two slots a compute unit; a stage takes 0.20 alone, 0.29 with one workgroup
// per compute unit, 0.60 with two, a workgroup 3.3 more. The widened products have this tile only, at 1.5 times
// its stage.
// So 8192 x 1280 x 5120 takes the 192 tile (224 of them: 57; 160 of 256: 62; 128: 77), 2048^3 the 128 tile (13
// against 28), and the two gradients of 8192 x 1280 -> 5120 together a large tile (128 against 162).
// A slice's partial sums are written and read again at some 4.5 TB/s and folded by a launch of 3: 1024 x 1024 x
// 8192 gains by four slices (33 -> 23), 2048^3 loses by two (13 -> 31).
struct Work {
  int64_t tasks;
  int steps;
};

static float time_stream(int tile, const Work* work, int n) {  // the longer tasks first
  const int64_t first = work[0].tasks, total = first + (n > 1 ? work[1].tasks : 0);
  const float load = total < kSlots ? total / float(kSlots) : 1.f;
  const float stage = tile == 256 ? 0.47f + 0.28f * load : 0.37f + 0.24f * load;
  auto task = [&](int64_t i) { return i >= total ? 0.f : 3.f + stage * work[i >= first].steps; };
  const int64_t rounds = ceil_div(total, kSlots);
  if (n == 1) return 10.f + rounds * task(0);
  if (rounds > 32) return 10.f + (first * task(0) + (total - first) * task(total - 1)) / kSlots + task(total - 1);
  float most = 0.f;
  for (int w = 0; w < kSlots; w += 15) {  // (0 and 255 among them)
    float t = 0.f;
    for (int64_t r = 0; r < rounds; ++r) t += task(r * kSlots + ((r & 1) ? kSlots - 1 - w : w));
    most = std::max(most, t);
  }
  return 10.f + most;
}

static float time_128(const Work* work, int n, bool wide) {
  const int64_t slots = 2 * kSlots;
  auto task = [&](int64_t tasks, int steps) {  // of so many at once
    const float load = std::min(tasks, slots) / float(kSlots);
    const float stage = load <= 1.f ? 0.20f + 0.09f * load : 0.29f + 0.31f * (load - 1.f);
    return 3.3f + steps * stage * (wide ? 1.5f : 1.f);
  };
  if (n == 1) {
    const int64_t full = work[0].tasks / slots, rest = work[0].tasks % slots;
    return 1.4f + full * task(slots, work[0].steps) + (rest ? task(rest, work[0].steps) : 0.f);
  }
  const int64_t total = work[0].tasks + work[1].tasks;
  const float a = task(total, work[0].steps), b = task(total, work[1].steps);
  if (total <= slots) return 1.4f + std::max(a, b);
  return 1.4f + (work[0].tasks * a + work[1].tasks * b) / slots + 0.5f * std::max(a, b);
}

// Up to two products that share a launch: one tile for both, each cut or not.
struct Choice {
  Fp8GemmPlan plan[2];
  float time;
};

// A tile is named by its features: 256 (and 256 tokens), 192 (256 tokens) or 128 (128 tokens).
static int64_t tiles_of(int tile, int M, int N) { return ceil_div(M, tile == 128 ? 128 : 256) * ceil_div(N, tile); }

static Work work_of(const Fp8GemmPlan& plan, const Fp8GemmProblem& p) {
  return Work{tiles_of(plan.tile, p.x.rows, p.w.rows) * plan.slices, std::min(plan.steps_per_slice, p.K / kStageK)};
}
static float fold_time(const Fp8GemmPlan& plan, const Fp8GemmProblem& p) {
  if (plan.slices == 1 && !p.accumulate) return 0.f;
  const float out = (p.out_dtype == kF32 ? 4.f : 2.f) * (p.accumulate ? 2.f : 1.f);
  return 3.f + float(p.x.rows) * p.w.rows * (8.f * plan.slices + out) / 4.5e6f;
}

// (of one launch: the problems are widened both or neither)
static float time_of(const Fp8GemmPlan* plans, const Fp8GemmProblem* problems, int n) {
  Work work[2] = {};
  float t = 0.f;
  for (int i = 0; i < n; ++i) {
    work[i] = work_of(plans[i], problems[i]);
    t += fold_time(plans[i], problems[i]);
  }
  if (n == 2 && work[1].steps > work[0].steps) std::swap(work[0], work[1]);
  return t + (plans[0].tile != 128 ? time_stream(plans[0].tile, work, n) : time_128(work, n, problems[0].out_dtype == kF32));
}

static Choice choose(int tile, const Fp8GemmProblem* problems, int n) {
  Choice best = {};
  Fp8GemmPlan whole[2], cut[2];
  for (int i = 0; i < n; ++i) {
    const int groups = (problems[i].K / kStageK + kGroupStages - 1) / kGroupStages;
    whole[i] = cut[i] = Fp8GemmPlan{tile, 1, groups * kGroupStages};
    float least = time_of(&whole[i], &problems[i], 1);
    for (int slices = 2; slices <= groups && slices <= 16; ++slices) {
      const int per = (groups + slices - 1) / slices;
      if ((groups + per - 1) / per != slices) continue;  // (a slice without work)
      const Fp8GemmPlan plan{tile, slices, per * kGroupStages};
      const float t = time_of(&plan, &problems[i], 1);
      if (t < least) least = t, cut[i] = plan;
    }
  }
  for (int k = 0; k < (1 << n); ++k) {
    Choice c = {};
    for (int i = 0; i < n; ++i) c.plan[i] = (k >> i) & 1 ? cut[i] : whole[i];
    c.time = time_of(c.plan, problems, n);
    if (k == 0 || c.time < best.time) best = c;
  }
  return best;
}

// No large tile: widened products, or what its epilogue's 32-bit offsets and bias loads do not reach.
static bool small_only(const Fp8GemmProblem& p) {
  return p.out_dtype == kF32 || p.w.rows > (1 << 20) || reinterpret_cast<uintptr_t>(p.bias) % 4 != 0;
}

// Two products share a launch, and so a tile, if they take the same kernel. Where they do not (a weight gradient into
// an fp32 buffer, which is widened and tied to the small tile, beside a bf16 input gradient), each is planned by itself.
void fp8_gemm_plan(Fp8GemmProblem* problems, int n) {
  auto alike = [&]() {
    return (problems[0].out_dtype == kF32) == (problems[1].out_dtype == kF32) && small_only(problems[0]) == small_only(problems[1]);
  };
  if (n == 2 && !alike()) {
    fp8_gemm_plan(problems, 1);
    fp8_gemm_plan(problems + 1, 1);
    return;
  }
  if (n == 0) return;
  Choice best = choose(128, problems, n);
  if (!small_only(problems[0])) {
    for (int tile : {192, 256}) {
      const Choice big = choose(tile, problems, n);
      if (big.time < best.time) best = big;
    }
  }
  for (int i = 0; i < n; ++i) problems[i].plan = best.plan[i];
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
    const int64_t tasks = tiles_of(g.plan.tile, M, N) * g.plan.slices;
    ps[i] = Problem{operand(g.x), operand(g.w), out, fold ? nullptr : g.bias, f32, g.bias_dtype == kF32,
                    g.K / kStageK, g.plan.steps_per_slice, (int)tasks};
    if (fold)
      add_fold(Fold{g.partial, g.bias, g.out, int64_t(M) * N, g.plan.slices, N, 0, g.bias_dtype == kF32, g.out_dtype == kF32,
                    g.accumulate, false});
  }
  auto go = [&](const Problem& a, const Problem* b, int tile, bool wide) {
    Problems P = {{a, b ? *b : Problem{}}};
    if (wide) launch<2, 2, true>(P, stream);
    else if (tile == 256) launch<4, 4, false>(P, stream);
    else if (tile == 192) launch<4, 3, false>(P, stream);
    else launch<2, 2, false>(P, stream);
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
