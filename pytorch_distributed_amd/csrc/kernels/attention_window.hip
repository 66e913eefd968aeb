// Causal attention inside a sliding window, with sink tokens, for gfx950: forward and backward.
//
//   query t sees key s  <=>  s <= t  and  (t - s < window  or  s < sinks)
//
// over the packed [B, T, 3, H, D] activation of the causal kernels (attention_common.h: layout, MFMA
// orientation, LDS swizzle), whose row and tile structure these share: a workgroup of 4 waves owns 128
// queries (dK / dV: keys), 32 per wave, and streams tiles of 64 keys (queries) through LDS. What the
// window changes:
//
//   forward, dQ   visit the tiles of the window from the diagonal down, then those that hold sinks. The
//                 first tile a wave works on is the one with its own diagonal, so every row has a finite
//                 running maximum from the first tile on, whatever later tiles mask.
//   dK, dV        a key is seen by `window` queries, a sink by all later ones. The main kernel streams the
//                 window's queries. The queries beyond it see a few sinks only: they are cut into chunks,
//                 each summed by a workgroup of its own into fp32 partials (launched first), which the main
//                 kernel's sums start from, added in chunk order. One workgroup for all queries of a sink
//                 would walk T / 64 tiles where the others walk window / 64 + 2.
//
// Every sum has one owner and a fixed order: results repeat bit for bit. Probabilities and their gradients
// are rounded to bf16 as operands of the second products (relative 2^-9 each, averaged by the sums); scores,
// softmax statistics and accumulators are fp32, and unlike the causal backward no operand is pre-scaled.
// Dropout draws the causal kernels' mask (a function of seed, head, query and key).
#include <type_traits>

#include "attention_common.h"
#include "pda_kernels.h"

namespace pda {
using attn::DropoutParams;
using attn::make_dropout_params;
namespace {

using namespace attn;

constexpr int kThreads = 256;
constexpr int kBM = 128;  // rows owned by a workgroup
constexpr int kBN = 64;   // rows per streamed tile

struct Shape {
  int B, T, H, window, sinks;
  float scale;
};

// The key tiles that queries q_first .. q_last (inclusive) of a workgroup visit: `n_win` tiles of the window
// downward from the diagonal's, then the tiles below them that hold sinks.
struct KeyTiles {
  int hi, n_win, n_sink, total;
  __device__ __forceinline__ KeyTiles(const Shape& s, int q_first, int q_last) {
    hi = q_last / kBN;
    const int lo = max(0, q_first - s.window + 1) / kBN;
    n_win = hi - lo + 1;
    n_sink = min(lo, (s.sinks + kBN - 1) / kBN);
    total = n_win + n_sink;
  }
  __device__ __forceinline__ int operator[](int i) const { return i < n_win ? hi - i : total - 1 - i; }
};

// How tile `key0` .. +63 meets the 32 queries from q0: nothing visible, some masked, or all visible.
// (The three tests are wave-uniform.)
__device__ __forceinline__ bool tile_seen(const Shape& s, int key0, int q0) {
  return key0 <= q0 + 31 && (key0 + kBN - 1 > q0 - s.window || key0 < s.sinks);
}
__device__ __forceinline__ bool tile_masked(const Shape& s, int key0, int q0) {
  return key0 + kBN - 1 > q0 || (q0 + 31 - key0 >= s.window && key0 + kBN > s.sinks);
}
__device__ __forceinline__ bool visible(const Shape& s, int q, int key) {
  return key <= q && (q - key < s.window || key < s.sinks);
}

// ======================================================================= forward
template <int D, bool kDrop>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 && !kDrop ? 3 : 2))) void window_fwd_kernel(
    const bf16_raw* __restrict__ qkv, bf16_raw* __restrict__ out, float* __restrict__ lse_out, Shape s, DropoutParams drop) {
  constexpr int kKSteps = D / 16;
  constexpr int kDBlocks = D / 32;
  constexpr int kTileBytes = kBN * D * 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // [2 buffers][K tile | V tile]

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;

  const int BH = s.B * s.H, T = s.T;
  const int bh = blockIdx.x % BH, qt = blockIdx.x / BH;
  const int b = bh / s.H, head = bh % s.H;
  const int64_t tok_stride = int64_t(3) * s.H * D;
  const bf16_raw* q_base = qkv + int64_t(b) * T * tok_stride + int64_t(head) * D;
  const bf16_raw* k_base = q_base + int64_t(s.H) * D;
  const bf16_raw* v_base = q_base + int64_t(2) * s.H * D;

  const int q0 = qt * kBM + wave * 32;
  const int q_row = q0 + r;
  const int q_ld = q_row < T ? q_row : T - 1;
  const bool wave_active = q0 < T;
  const KeyTiles tiles(s, qt * kBM, min(qt * kBM + kBM, T) - 1);

  TileStager<D, kBN, kThreads> k_stage, v_stage;
  k_stage.load(k_base, tok_stride, tiles[0] * kBN, T - 1, tid);
  v_stage.load(v_base, tok_stride, tiles[0] * kBN, T - 1, tid);
  bf16x8 qf[kKSteps];
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks)
    qf[ks] = *reinterpret_cast<const bf16x8*>(q_base + int64_t(q_ld) * tok_stride + 16 * ks + 8 * h);

  f32x16 o_acc[kDBlocks];
#pragma unroll
  for (int i = 0; i < kDBlocks; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o_acc[i][j] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;  // running row maximum (exp2 units), this lane's share of the row sum
  const float c = s.scale * kLog2e;

  k_stage.store(smem, tid);
  v_stage.store(smem + kTileBytes, tid);
  // Q has arrived here, not at its first use inside the loop, where the wait would include the prefetch
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) asm volatile("" ::"v"(__builtin_bit_cast(u32x4, qf[ks])));
  __syncthreads();

  for (int j = 0; j < tiles.total; ++j) {
    const char* k_tile = smem + (j & 1) * 2 * kTileBytes;
    const char* v_tile = k_tile + kTileBytes;
    const int key0 = tiles[j] * kBN;
    const bool has_next = j + 1 < tiles.total;
    if (has_next) {
      k_stage.load(k_base, tok_stride, tiles[j + 1] * kBN, T - 1, tid);
      v_stage.load(v_base, tok_stride, tiles[j + 1] * kBN, T - 1, tid);
    }

    if (wave_active && tile_seen(s, key0, q0)) {
      f32x16 s_acc[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s_acc[kb][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < kKSteps; ++ks) {
          const bf16x8 kf = lds_read_b128(k_tile, tile_off<D>(kb * 32 + r, 2 * ks + h));
          s_acc[kb] = mfma32(kf, qf[ks], s_acc[kb]);
        }
      }
      // max3() is inline assembly behind a matrix instruction: the wait states are explicit
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s_acc[0]), "+v"(s_acc[1]));
      auto row_max = [&](auto masked) {
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          if (decltype(masked)::value) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!visible(s, q_row, key0 + kb * 32 + acc_row(i + e, h))) s_acc[kb][i + e] = -INFINITY;
          }
          m0 = max3(m0, s_acc[0][i], s_acc[0][i + 1]);
          m1 = max3(m1, s_acc[1][i], s_acc[1][i + 1]);
        }
        return fmaxf(m0, m1);
      };
      float mx;
      if (tile_masked(s, key0, q0)) mx = row_max(std::true_type{});  // wave-uniform
      else mx = row_max(std::false_type{});
      mx = c * lane_pair_max(mx);
      const float m_new = fmaxf(m_run, mx);  // finite: the wave's first tile holds every row's own key
      const bool grew = m_new > m_run;
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      float psum0 = 0.f, psum1 = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          s_acc[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s_acc[kb][i], c, -m_new));
          s_acc[kb][i + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s_acc[kb][i + 1], c, -m_new));
          psum0 += s_acc[kb][i];
          psum1 += s_acc[kb][i + 1];
        }
      l_run = l_run * alpha + (psum0 + psum1);
      if (__builtin_amdgcn_ballot_w64(grew) != 0) {  // wave-uniform
#pragma unroll
        for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o_acc[db][i] *= alpha;
      }
      if (kDrop) {  // the row sum is of the undropped probabilities
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t words[4];
          dropout_words_for_query(drop, bh, q_row, key0 + kb * 32, h, lane, words);
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool keep = ((words[g] >> (8 * e)) & 0xffu) >= drop.threshold;
              s_acc[kb][4 * g + e] = keep ? s_acc[kb][4 * g + e] * drop.keep_scale : 0.f;
            }
        }
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const f32x16& p = s_acc[ks >> 1];
        const int o = 8 * (ks & 1);
        const bf16x8 pf = pack_acc8(p[o], p[o + 1], p[o + 2], p[o + 3], p[o + 4], p[o + 5], p[o + 6], p[o + 7]);
#pragma unroll
        for (int db = 0; db < kDBlocks; ++db) o_acc[db] = mfma32(tr_fragment<D>(v_tile, ks, db, lane), pf, o_acc[db]);
      }
    }

    if (has_next) {
      char* nk = smem + ((j + 1) & 1) * 2 * kTileBytes;
      k_stage.store(nk, tid);
      v_stage.store(nk + kTileBytes, tid);
    }
    __syncthreads();
  }

  const float l_tot = lane_pair_sum(l_run);
  if (q_row < T) {
    const float inv_l = 1.f / l_tot;
    bf16_raw* o_row = out + (int64_t(b) * T + q_row) * (int64_t(s.H) * D) + int64_t(head) * D;
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 w = {pack_bf16x2(o_acc[db][4 * g] * inv_l, o_acc[db][4 * g + 1] * inv_l),
                   pack_bf16x2(o_acc[db][4 * g + 2] * inv_l, o_acc[db][4 * g + 3] * inv_l)};
        *reinterpret_cast<u32x2*>(o_row + db * 32 + 8 * g + 4 * h) = w;
      }
    // log2 of the row's sum of exponentials (the backward's exponent offset)
    if (h == 0) lse_out[int64_t(bh) * T + q_row] = m_run + __log2f(l_tot);
  }
}

// ============================================================================ dQ
// S^T = K Q^T, P^T = exp2(c S^T - lse), dP^T = V dO^T, dS^T = P^T (dP^T - delta), dQ^T += K^T dS^T;
// also delta = rowsum(dO O) for the dK / dV kernels.
template <int D, bool kDrop>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1))) void window_dq_kernel(
    const bf16_raw* __restrict__ qkv, const bf16_raw* __restrict__ out, const bf16_raw* __restrict__ dout,
    const float* __restrict__ lse, float* __restrict__ delta_out, bf16_raw* __restrict__ dqkv, Shape s, DropoutParams drop) {
  constexpr int kKSteps = D / 16;
  constexpr int kDBlocks = D / 32;
  constexpr int kTileBytes = kBN * D * 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;

  const int BH = s.B * s.H, T = s.T;
  const int bh = blockIdx.x % BH, qt = blockIdx.x / BH;
  const int b = bh / s.H, head = bh % s.H;
  const int64_t tok_stride = int64_t(3) * s.H * D, o_stride = int64_t(s.H) * D;
  const bf16_raw* q_base = qkv + int64_t(b) * T * tok_stride + int64_t(head) * D;
  const bf16_raw* k_base = q_base + int64_t(s.H) * D;
  const bf16_raw* v_base = q_base + int64_t(2) * s.H * D;

  const int q0 = qt * kBM + wave * 32;
  const int q_row = q0 + r;
  const int q_ld = q_row < T ? q_row : T - 1;
  const bool wave_active = q0 < T;
  const KeyTiles tiles(s, qt * kBM, min(qt * kBM + kBM, T) - 1);

  TileStager<D, kBN, kThreads> k_stage, v_stage;
  k_stage.load(k_base, tok_stride, tiles[0] * kBN, T - 1, tid);
  v_stage.load(v_base, tok_stride, tiles[0] * kBN, T - 1, tid);

  bf16x8 qf[kKSteps], dof[kKSteps];
  float dpart = 0.f;
  {
    const bf16_raw* o_row = out + (int64_t(b) * T + q_ld) * o_stride + int64_t(head) * D;
    const bf16_raw* do_row = dout + (int64_t(b) * T + q_ld) * o_stride + int64_t(head) * D;
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      qf[ks] = *reinterpret_cast<const bf16x8*>(q_base + int64_t(q_ld) * tok_stride + 16 * ks + 8 * h);
      dof[ks] = *reinterpret_cast<const bf16x8*>(do_row + 16 * ks + 8 * h);
      const bf16x8 of = *reinterpret_cast<const bf16x8*>(o_row + 16 * ks + 8 * h);
#pragma unroll
      for (int j = 0; j < 8; ++j) dpart += (float)dof[ks][j] * (float)of[j];
    }
  }
  const float delta = lane_pair_sum(dpart);
  const float neg_lse = -lse[int64_t(bh) * T + q_ld];
  if (h == 0 && q_row < T) delta_out[int64_t(bh) * T + q_row] = delta;
  const float c = s.scale * kLog2e;

  f32x16 dq_acc[kDBlocks];
#pragma unroll
  for (int i = 0; i < kDBlocks; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) dq_acc[i][j] = 0.f;

  k_stage.store(smem, tid);
  v_stage.store(smem + kTileBytes, tid);
  __syncthreads();

  for (int j = 0; j < tiles.total; ++j) {
    const char* k_tile = smem + (j & 1) * 2 * kTileBytes;
    const char* v_tile = k_tile + kTileBytes;
    const int key0 = tiles[j] * kBN;
    const bool has_next = j + 1 < tiles.total;
    if (has_next) {
      k_stage.load(k_base, tok_stride, tiles[j + 1] * kBN, T - 1, tid);
      v_stage.load(v_base, tok_stride, tiles[j + 1] * kBN, T - 1, tid);
    }

    if (wave_active && tile_seen(s, key0, q0)) {
      f32x16 s_acc[2], dp_acc[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s_acc[kb][i] = 0.f;
          dp_acc[kb][i] = -delta;  // the chain ends as dP - delta
        }
      // fragments are requested half a tile ahead of the products that take them
      bf16x8 frag[2][2 * kKSteps];
      auto request = [&](int kb, int i) {
        frag[kb][i] = lds_read_b128(i < kKSteps ? k_tile : v_tile, tile_off<D>(kb * 32 + r, 2 * (i % kKSteps) + h));
      };
      auto multiply = [&](int kb, int i) {
        if (i < kKSteps) s_acc[kb] = mfma32(frag[kb][i], qf[i], s_acc[kb]);
        else dp_acc[kb] = mfma32(frag[kb][i], dof[i - kKSteps], dp_acc[kb]);
      };
#pragma unroll
      for (int i = 0; i < 2 * kKSteps; ++i) request(0, i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * kKSteps; ++i) {
        multiply(0, i);
        request(1, i);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 2 * kKSteps; ++i) multiply(1, i);
      __builtin_amdgcn_sched_barrier(0);

      if (kDrop) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t words[4];
          dropout_words_for_query(drop, bh, q_row, key0 + kb * 32, h, lane, words);
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool keep = ((words[g] >> (8 * e)) & 0xffu) >= drop.threshold;
              const float dp_true = dp_acc[kb][4 * g + e] + delta;
              dp_acc[kb][4 * g + e] = (keep ? dp_true * drop.keep_scale : 0.f) - delta;
            }
        }
      }
      auto softmax_grad = [&](auto masked) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s_acc[kb][i], c, neg_lse));
            if (decltype(masked)::value)
              if (!visible(s, q_row, key0 + kb * 32 + acc_row(i, h))) p = 0.f;
            s_acc[kb][i] = p * dp_acc[kb][i];
          }
      };
      if (tile_masked(s, key0, q0)) softmax_grad(std::true_type{});
      else softmax_grad(std::false_type{});
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const f32x16& a = s_acc[ks >> 1];
        const int o = 8 * (ks & 1);
        const bf16x8 dsf = pack_acc8(a[o], a[o + 1], a[o + 2], a[o + 3], a[o + 4], a[o + 5], a[o + 6], a[o + 7]);
#pragma unroll
        for (int db = 0; db < kDBlocks; ++db) dq_acc[db] = mfma32(tr_fragment<D>(k_tile, ks, db, lane), dsf, dq_acc[db]);
      }
    }

    if (has_next) {
      char* nk = smem + ((j + 1) & 1) * 2 * kTileBytes;
      k_stage.store(nk, tid);
      v_stage.store(nk + kTileBytes, tid);
    }
    __syncthreads();
  }

  if (q_row < T) {
    bf16_raw* dq_row = dqkv + (int64_t(b) * T + q_row) * tok_stride + int64_t(head) * D;
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 w = {pack_bf16x2(dq_acc[db][4 * g] * s.scale, dq_acc[db][4 * g + 1] * s.scale),
                   pack_bf16x2(dq_acc[db][4 * g + 2] * s.scale, dq_acc[db][4 * g + 3] * s.scale)};
        *reinterpret_cast<u32x2*>(dq_row + db * 32 + 8 * g + 4 * h) = w;
      }
  }
}

// ========================================================================= dK / dV
// Partial sums of the queries beyond the window, for the first `rows` (sinks rounded up to 32) keys:
// fp32 [B * H][chunks][2: dK, dV][rows][D]. kFar: chunk blockIdx / (BH * key tiles) of those queries.
struct FarSums {
  float* ptr;
  int chunks, tiles_per_chunk, rows;
};

template <int D, bool kDrop, bool kFar>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1))) void window_dkv_kernel(
    const bf16_raw* __restrict__ qkv, const bf16_raw* __restrict__ dout, const float* __restrict__ lse,
    const float* __restrict__ delta, bf16_raw* __restrict__ dqkv, FarSums far, Shape s, DropoutParams drop) {
  constexpr int kKSteps = D / 16;
  constexpr int kDBlocks = D / 32;
  constexpr int kTileBytes = kBN * D * 2;
  // [2][Q tile | dO tile], then [2][64 x (-lse) | 64 x (-delta)] fp32 row constants
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* rowc = reinterpret_cast<float*>(smem + 4 * kTileBytes);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;

  const int BH = s.B * s.H, T = s.T;
  const int bh = blockIdx.x % BH;
  const int n_sink_tiles = (far.rows + kBM - 1) / kBM;
  const int kt = kFar ? (blockIdx.x / BH) % n_sink_tiles : blockIdx.x / BH;
  const int chunk = kFar ? blockIdx.x / (BH * n_sink_tiles) : 0;
  const int b = bh / s.H, head = bh % s.H;
  const int64_t tok_stride = int64_t(3) * s.H * D, o_stride = int64_t(s.H) * D;
  const bf16_raw* q_base = qkv + int64_t(b) * T * tok_stride + int64_t(head) * D;
  const bf16_raw* k_base = q_base + int64_t(s.H) * D;
  const bf16_raw* v_base = q_base + int64_t(2) * s.H * D;
  const bf16_raw* do_base = dout + int64_t(b) * T * o_stride + int64_t(head) * D;
  const float* lse_row = lse + int64_t(bh) * T;
  const float* delta_row = delta + int64_t(bh) * T;

  const int key0 = kt * kBM + wave * 32;  // first key of this wave
  const int key = key0 + r;               // this lane's key
  const int key_ld = key < T ? key : T - 1;
  const bool wave_active = kFar ? key0 < far.rows : key0 < T;

  // Query tiles: the window's (from the diagonal to the last query that sees the last key), or this chunk's
  // share of those beyond it.
  const int n_tiles = (T + kBN - 1) / kBN;
  int first_tile, end_tile;
  if (kFar) {
    first_tile = (kt * kBM + s.window) / kBN + chunk * far.tiles_per_chunk;
    end_tile = min(n_tiles, first_tile + far.tiles_per_chunk);
  } else {
    first_tile = kt * kBM / kBN;
    // (window may be as large as an int: compare before adding)
    const int last_q = s.window > T ? T - 1 : min(T - 1, kt * kBM + kBM - 1 + s.window - 1);
    end_tile = last_q / kBN + 1;
  }

  bf16x8 kf[kKSteps], vf[kKSteps];
  f32x16 dk_acc[kDBlocks], dv_acc[kDBlocks];
#pragma unroll
  for (int i = 0; i < kDBlocks; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      dk_acc[i][j] = 0.f;
      dv_acc[i][j] = 0.f;
    }
  // Keys that are sinks start from the far queries' sums, added in chunk order. (Lane (r, h) holds elements
  // 32 db + 8 g + 4 h .. +3 of key r's rows.)
  if (!kFar && key0 < far.rows) {  // wave-uniform
    for (int ch = 0; ch < far.chunks; ++ch) {
      const float* dk_row = far.ptr + ((int64_t(bh) * far.chunks + ch) * 2 * far.rows + key) * D;
      const float* dv_row = dk_row + int64_t(far.rows) * D;
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int o = db * 32 + 8 * g + 4 * h;
          const f32x4 a = *reinterpret_cast<const f32x4*>(dk_row + o), d = *reinterpret_cast<const f32x4*>(dv_row + o);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dk_acc[db][4 * g + e] += a[e];
            dv_acc[db][4 * g + e] += d[e];
          }
        }
    }
  }
  const float c = s.scale * kLog2e;

  if (first_tile < end_tile) {  // workgroup-uniform (a key tile of the far part can have no query left)
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      kf[ks] = *reinterpret_cast<const bf16x8*>(k_base + int64_t(key_ld) * tok_stride + 16 * ks + 8 * h);
      vf[ks] = *reinterpret_cast<const bf16x8*>(v_base + int64_t(key_ld) * tok_stride + 16 * ks + 8 * h);
    }
    const float* rowc_src = tid < 64 ? lse_row : delta_row;
    auto load_rowc = [&](int tile) -> float {
      if (tid >= 128) return 0.f;
      int q = tile * kBN + (tid & 63);
      q = q < T ? q : T - 1;
      return rowc_src[q];
    };
    TileStager<D, kBN, kThreads> q_stage, do_stage;
    q_stage.load(q_base, tok_stride, first_tile * kBN, T - 1, tid);
    do_stage.load(do_base, o_stride, first_tile * kBN, T - 1, tid);
    float rc_stage = load_rowc(first_tile);
    // K and V have arrived here, not at their first use inside the loop
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      asm volatile("" ::"v"(__builtin_bit_cast(u32x4, kf[ks])));
      asm volatile("" ::"v"(__builtin_bit_cast(u32x4, vf[ks])));
    }
    q_stage.store(smem, tid);
    do_stage.store(smem + kTileBytes, tid);
    if (tid < 128) rowc[tid] = -rc_stage;
    __syncthreads();

    for (int j = first_tile; j < end_tile; ++j) {
      const int buf = (j - first_tile) & 1;
      const char* q_tile = smem + buf * 2 * kTileBytes;
      const char* do_tile = q_tile + kTileBytes;
      const bool has_next = j + 1 < end_tile;
      const float* rc = rowc + buf * 128;
      if (has_next) {
        q_stage.load(q_base, tok_stride, (j + 1) * kBN, T - 1, tid);
        do_stage.load(do_base, o_stride, (j + 1) * kBN, T - 1, tid);
        rc_stage = load_rowc(j + 1);
      }

      if (wave_active) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {  // two 32-query sub-tiles
          const int qs = j * kBN + sub * 32;
          // wave-uniform: nothing of this sub-tile belongs to this wave's keys
          const bool none = kFar ? qs + 31 - key0 < s.window || qs >= T
                                 : qs + 31 < key0 || qs >= T || qs - (key0 + 31) >= s.window;
          if (none) continue;
          f32x16 s_acc, dp_acc;
          float neg_lse[16];
          float neg_delta[kDrop ? 16 : 1];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(rc + sub * 32 + 8 * g + 4 * h);
            const f32x4 d = *reinterpret_cast<const f32x4*>(rc + 64 + sub * 32 + 8 * g + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s_acc[4 * g + e] = 0.f;
              neg_lse[4 * g + e] = a[e];
              dp_acc[4 * g + e] = d[e];  // the chain ends as dP - delta
              if (kDrop) neg_delta[4 * g + e] = d[e];
            }
          }
#pragma unroll
          for (int ks = 0; ks < kKSteps; ++ks)
            s_acc = mfma32(lds_read_b128(q_tile, tile_off<D>(sub * 32 + r, 2 * ks + h)), kf[ks], s_acc);
#pragma unroll
          for (int ks = 0; ks < kKSteps; ++ks)
            dp_acc = mfma32(lds_read_b128(do_tile, tile_off<D>(sub * 32 + r, 2 * ks + h)), vf[ks], dp_acc);
          uint32_t keep_mask = 0xffffu;
          if (kDrop) keep_mask = dropout_keep_mask_for_key(drop, bh, qs, h, key, lane);
          auto softmax_grad = [&](auto masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s_acc[i], c, neg_lse[i]));
              if (decltype(masked)::value) {
                const int q = qs + acc_row(i, h);
                const bool mine = kFar ? q - key >= s.window && key < s.sinks : q >= key && q - key < s.window;
                if (!mine || q >= T) p = 0.f;
              }
              if (kDrop) {
                const bool keep = (keep_mask >> i) & 1;
                const float dp = (keep ? (dp_acc[i] - neg_delta[i]) * drop.keep_scale : 0.f) + neg_delta[i];
                dp_acc[i] = p * dp;
                s_acc[i] = keep ? p * drop.keep_scale : 0.f;
              } else {
                s_acc[i] = p;
                dp_acc[i] = p * dp_acc[i];
              }
            }
          };
          const bool edge = kFar ? qs - (key0 + 31) < s.window || key0 + 32 > s.sinks
                                 : qs < key0 + 31 || qs + 31 - key0 >= s.window;
          if (edge || qs + 31 >= T) softmax_grad(std::true_type{});  // wave-uniform
          else softmax_grad(std::false_type{});
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int o = 8 * k;
            const bf16x8 pf = pack_acc8(s_acc[o], s_acc[o + 1], s_acc[o + 2], s_acc[o + 3], s_acc[o + 4], s_acc[o + 5],
                                        s_acc[o + 6], s_acc[o + 7]);
            const bf16x8 dsf = pack_acc8(dp_acc[o], dp_acc[o + 1], dp_acc[o + 2], dp_acc[o + 3], dp_acc[o + 4],
                                         dp_acc[o + 5], dp_acc[o + 6], dp_acc[o + 7]);
#pragma unroll
            for (int db = 0; db < kDBlocks; ++db) {
              dv_acc[db] = mfma32(tr_fragment<D>(do_tile, 2 * sub + k, db, lane), pf, dv_acc[db]);
              dk_acc[db] = mfma32(tr_fragment<D>(q_tile, 2 * sub + k, db, lane), dsf, dk_acc[db]);
            }
          }
        }
      }

      if (has_next) {
        char* nq = smem + (buf ^ 1) * 2 * kTileBytes;
        q_stage.store(nq, tid);
        do_stage.store(nq + kTileBytes, tid);
        if (tid < 128) rowc[(buf ^ 1) * 128 + tid] = -rc_stage;
      }
      __syncthreads();
    }
  }

  if (kFar) {
    if (!wave_active) return;  // no barrier follows
    float* dk_row = far.ptr + ((int64_t(bh) * far.chunks + chunk) * 2 * far.rows + key) * D;
    float* dv_row = dk_row + int64_t(far.rows) * D;
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int o = db * 32 + 8 * g + 4 * h;
        *reinterpret_cast<f32x4*>(dk_row + o) = f32x4{dk_acc[db][4 * g], dk_acc[db][4 * g + 1], dk_acc[db][4 * g + 2], dk_acc[db][4 * g + 3]};
        *reinterpret_cast<f32x4*>(dv_row + o) = f32x4{dv_acc[db][4 * g], dv_acc[db][4 * g + 1], dv_acc[db][4 * g + 2], dv_acc[db][4 * g + 3]};
      }
    return;
  }
  if (key < T) {
    bf16_raw* dk_row = dqkv + (int64_t(b) * T + key) * tok_stride + int64_t(s.H) * D + int64_t(head) * D;
    bf16_raw* dv_row = dk_row + int64_t(s.H) * D;
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 wk = {pack_bf16x2(dk_acc[db][4 * g] * s.scale, dk_acc[db][4 * g + 1] * s.scale),
                    pack_bf16x2(dk_acc[db][4 * g + 2] * s.scale, dk_acc[db][4 * g + 3] * s.scale)};
        u32x2 wv = {pack_bf16x2(dv_acc[db][4 * g], dv_acc[db][4 * g + 1]),
                    pack_bf16x2(dv_acc[db][4 * g + 2], dv_acc[db][4 * g + 3])};
        *reinterpret_cast<u32x2*>(dk_row + db * 32 + 8 * g + 4 * h) = wk;
        *reinterpret_cast<u32x2*>(dv_row + db * 32 + 8 * g + 4 * h) = wv;
      }
  }
}

// The far part's chunks: enough workgroups for two per compute unit, at least four query tiles each.
FarSums far_plan(int B, int T, int H, int window, int sinks) {
  FarSums f{nullptr, 0, 0, 0};
  if (sinks <= 0 || window >= T) return f;
  const int last_sink = sinks < T ? sinks : T;
  f.rows = (last_sink + 31) / 32 * 32;
  const int tiles = (T + kBN - 1) / kBN - window / kBN;  // from the first query beyond the window
  const int64_t owners = int64_t(B) * H * ((f.rows + kBM - 1) / kBM);
  int chunks = (int)((512 + owners - 1) / owners);
  const int most = (tiles + 3) / 4;
  if (chunks > most) chunks = most;
  f.tiles_per_chunk = (tiles + chunks - 1) / chunks;
  f.chunks = (tiles + f.tiles_per_chunk - 1) / f.tiles_per_chunk;
  return f;
}

}  // namespace

void window_attention_forward(const void* qkv, void* out, float* lse, int B, int T, int H, int D, int window, int sinks,
                              float softmax_scale, float dropout_p, uint64_t seed, hipStream_t stream) {
  const Shape s{B, T, H, window, sinks, softmax_scale};
  const dim3 grid((unsigned)(ceil_div(T, kBM) * B * H)), block(kThreads);
  const DropoutParams drop = make_dropout_params(dropout_p, seed);
  const size_t lds = size_t(2) * 2 * kBN * D * 2;
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, block, lds, stream, (const bf16_raw*)qkv, (bf16_raw*)out, lse, s, drop);
  };
  if (D == 64) {
    if (drop.threshold) launch(window_fwd_kernel<64, true>);
    else launch(window_fwd_kernel<64, false>);
  } else {
    if (drop.threshold) launch(window_fwd_kernel<128, true>);
    else launch(window_fwd_kernel<128, false>);
  }
}

size_t window_attention_backward_workspace_bytes(int B, int T, int H, int D, int window, int sinks) {
  const FarSums f = far_plan(B, T, H, window, sinks);
  return size_t(B) * H * f.chunks * 2 * f.rows * D * sizeof(float);
}

void window_attention_backward(const void* qkv, const void* out, const void* dout, const float* lse, float* delta,
                               void* dqkv, void* workspace, int B, int T, int H, int D, int window, int sinks,
                               float softmax_scale, float dropout_p, uint64_t seed, hipStream_t stream) {
  const Shape s{B, T, H, window, sinks, softmax_scale};
  FarSums far = far_plan(B, T, H, window, sinks);
  far.ptr = (float*)workspace;
  const dim3 grid((unsigned)(ceil_div(T, kBM) * B * H)), block(kThreads);
  const dim3 far_grid((unsigned)(ceil_div(far.rows, kBM) * far.chunks * B * H));
  const DropoutParams drop = make_dropout_params(dropout_p, seed);
  const size_t lds = size_t(2) * 2 * kBN * D * 2;
  auto launch = [&](auto dq_kern, auto far_kern, auto dkv_kern) {
    hipLaunchKernelGGL(dq_kern, grid, block, lds, stream, (const bf16_raw*)qkv, (const bf16_raw*)out, (const bf16_raw*)dout,
                       lse, delta, (bf16_raw*)dqkv, s, drop);
    if (far.chunks > 0)
      hipLaunchKernelGGL(far_kern, far_grid, block, lds + 1024, stream, (const bf16_raw*)qkv, (const bf16_raw*)dout, lse,
                         delta, (bf16_raw*)dqkv, far, s, drop);
    hipLaunchKernelGGL(dkv_kern, grid, block, lds + 1024, stream, (const bf16_raw*)qkv, (const bf16_raw*)dout, lse, delta,
                       (bf16_raw*)dqkv, far, s, drop);
  };
  if (D == 64) {
    if (drop.threshold) launch(window_dq_kernel<64, true>, window_dkv_kernel<64, true, true>, window_dkv_kernel<64, true, false>);
    else launch(window_dq_kernel<64, false>, window_dkv_kernel<64, false, true>, window_dkv_kernel<64, false, false>);
  } else {
    if (drop.threshold) launch(window_dq_kernel<128, true>, window_dkv_kernel<128, true, true>, window_dkv_kernel<128, true, false>);
    else launch(window_dq_kernel<128, false>, window_dkv_kernel<128, false, true>, window_dkv_kernel<128, false, false>);
  }
}

}  // namespace pda
