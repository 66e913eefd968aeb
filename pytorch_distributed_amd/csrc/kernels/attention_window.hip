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
// Tiles travel global -> LDS by buffer loads that write LDS directly (no registers on the way), one tile ahead
// of the products and issued one at a time between them, one barrier per tile. All LDS reads are inline assembly:
// the compiler cannot tell them from the destination of those loads and would wait for every load in flight before
// each of them. Each read is requested kAhead products before the one that takes it and awaited by count.
//
// What bounds them: latency, hidden by as many waves as the registers allow. 1 x 8192, 32 heads of 128, window 1024,
// 4 sinks: forward 201 us (matrix pipes 31 % busy, two waves on a SIMD), dQ 262 (38 %; at one wave 361), dK / dV 350
// and 44 for the far sinks. 8 x 1024, 20 heads of 64, window 256: forward 33 us (four waves; at three 40; 37 with the
// rest for the backward), dQ 47, dK / dV 42 (three waves each); there the vector unit's exponentials weigh as much
// as the products. Results leave through LDS in whole rows (dK / dV 48 -> 43 there).
//
// Every sum has one owner and a fixed order: results repeat bit for bit. Probabilities and their gradients
// are rounded to bf16 as operands of the second products (by at most 2^-8 of each, averaged by the sums); scores,
// softmax statistics and accumulators are fp32, and unlike the causal backward no operand is pre-scaled.
// Dropout draws the causal kernels' mask (a function of seed, head, query and key).
#include "attention_window.h"

namespace pda {
using attn::DropoutParams;
using attn::make_dropout_params;
namespace {

using namespace window;

// What bf16 drops of O, for delta = rowsum(dO O) (see window_dq_kernel): four values as e5m2 times 2^9, which
// puts the rest of a value of size |o| near |o| itself. Values whose rest leaves e5m2's range lose it or clamp.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, float c, float d) {
  auto fit = [](float v) { return __builtin_fminf(__builtin_fmaxf(v * 512.f, -57344.f), 57344.f); };
  const int w = __builtin_amdgcn_cvt_pk_bf8_f32(fit(a), fit(b), 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_bf8_f32(fit(c), fit(d), w, true));
}
__device__ __forceinline__ void unpack_rest(u32x2 w, float (&out)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_bf8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_bf8((int)w[i], true);
    out[4 * i] = a[0] * (1.f / 512.f);
    out[4 * i + 1] = a[1] * (1.f / 512.f);
    out[4 * i + 2] = b[0] * (1.f / 512.f);
    out[4 * i + 3] = b[1] * (1.f / 512.f);
  }
}

// ======================================================================= forward
template <int D, bool kDrop>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? (kDrop ? 3 : 4) : 2))) void window_fwd_kernel(
    const bf16_raw* __restrict__ qkv, bf16_raw* __restrict__ out, uint8_t* __restrict__ out_rest,
    float* __restrict__ neg_lse_out, Shape s, DropoutParams drop) {
  constexpr int kKSteps = D / 16;
  constexpr int kDBlocks = D / 32;
  constexpr int kTileBytes = kBN * D * 2;
  constexpr int kAhead = D == 64 ? 4 : 6, kAheadV = D == 64 ? 2 : 3;  // row reads / transposed fragments in flight
  extern __shared__ __attribute__((aligned(16))) char smem[];  // [2 buffers][K tile | V tile]

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

  TileLoader<D> loader;
  loader.init(tok_stride, wave, lane);
  loader.load(k_base, tiles[0] * kBN, T - 1, smem, wave);
  loader.load(v_base, tiles[0] * kBN, T - 1, smem + kTileBytes, wave);
  auto following = [&](int j) {  // tile j + 1 (behind the last: nothing)
    const bool more = j + 1 < tiles.total;
    const int first = tiles[more ? j + 1 : j] * kBN, last = more ? T - 1 : -1;
    return NextTile<D>{loader.aim(k_base, first, last), loader.aim(v_base, first, last), smem + ((j + 1) & 1) * 2 * kTileBytes};
  };
  bf16x8 qf[kKSteps];
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks)
    qf[ks] = *reinterpret_cast<const bf16x8*>(q_base + int64_t(q_ld) * tok_stride + 16 * ks + 8 * h);
  // Q arrives here, beside the first tile, not at its first use inside the loop, where the wait would include the
  // next tile
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) asm volatile("" ::"v"(__builtin_bit_cast(u32x4, qf[ks])));
  TileAddr<D> at;
  at.init(lds_addr(smem), lane);

  f32x16 o_acc[kDBlocks];
#pragma unroll
  for (int i = 0; i < kDBlocks; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o_acc[i][j] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;  // running reference of the row (exp2 units), this lane's share of the row sum
  const float c = s.scale * kLog2e;

  for (int j = 0; j < tiles.total; ++j) {
    const int key0 = tiles[j] * kBN;
    next_tile_ready();
    const NextTile<D> next = following(j);

    if (wave_active && tile_seen(s, key0, q0)) {
      u32x4 kf[kAhead];
      auto request = [&](auto n) {  // product n: step n / 2 of key half n % 2
        kf[n % kAhead] = read16<(n % 2) * 64 * D>(at.row[n / 2]);
      };
      constexpr int kN = 2 * kKSteps;
      static_for<0, kAhead>(request);
      f32x16 s_acc[2];
      float first[2][16] = {};
      if (tile_masked(s, key0, q0)) {  // wave-uniform
        start_masked(s, q_row, key0, h, first[0]);
        start_masked(s, q_row, key0 + 32, h, first[1]);
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s_acc[kb][i] = first[kb][i];
      static_for<0, kN>([&](auto n) {
        constexpr int kb = n % 2, ks = n / 2;
        wait_for<(kN - 1 - n < kAhead - 1 ? kN - 1 - n : kAhead - 1)>(kf[n % kAhead]);
        s_acc[kb] = mfma32(__builtin_bit_cast(bf16x8, kf[n % kAhead]), qf[ks], s_acc[kb]);
        if constexpr (n + kAhead < kN) request(std::integral_constant<int, n + kAhead>{});
        next.template behind<n>(loader, loader, wave);
        __builtin_amdgcn_sched_barrier(0);
      });
      // the first V fragments travel under the softmax
      constexpr int kVN = 4 * kDBlocks;  // fragment n: 16-key step n / kDBlocks, column block n % kDBlocks
      u32x2 vlo[kAheadV], vhi[kAheadV];
      auto request_v = [&](auto n) {
        constexpr int k = n / kDBlocks, db = n % kDBlocks;
        vlo[n % kAheadV] = read_tr8<kTileBytes + k * 32 * D>(at.tr[db][0]);
        vhi[n % kAheadV] = read_tr8<kTileBytes + k * 32 * D>(at.tr[db][1]);
      };
      static_for<0, kAheadV>(request_v);
      __builtin_amdgcn_sched_barrier(0);
      // max3() is inline assembly behind a matrix instruction: the wait states are explicit
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s_acc[0]), "+v"(s_acc[1]));
      float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        m0 = max3(m0, s_acc[0][i], s_acc[0][i + 1]);
        m1 = max3(m1, s_acc[1][i], s_acc[1][i + 1]);
      }
      float mx = fmaxf(m0, m1);
      mx = c * lane_pair_max(mx);
      // A row's reference moves only when its maximum has outgrown it by 2^8: probabilities up to 256 times the
      // reference's cost no precision, and most tiles are spared the pass over the accumulators (with 32 rows to a
      // wave, nearly every tile has some row with a new maximum).
      const bool grew = mx > m_run + 8.f;
      const float m_new = grew ? mx : m_run;  // finite: the wave's first tile holds every row's own key
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
      bf16x8 pf[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x16& p = s_acc[k >> 1];
        const int o = 8 * (k & 1);
        pf[k] = pack_acc8(p[o], p[o + 1], p[o + 2], p[o + 3], p[o + 4], p[o + 5], p[o + 6], p[o + 7]);
      }
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, kVN>([&](auto n) {
        constexpr int left = kVN - 1 - n < kAheadV - 1 ? kVN - 1 - n : kAheadV - 1;
        wait_for<2 * left>(vlo[n % kAheadV], vhi[n % kAheadV]);
        o_acc[n % kDBlocks] = mfma32(join(vlo[n % kAheadV], vhi[n % kAheadV]), pf[n / kDBlocks], o_acc[n % kDBlocks]);
        if constexpr (n + kAheadV < kVN) request_v(std::integral_constant<int, n + kAheadV>{});
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      static_for<0, NextTile<D>::kLoads>([&](auto i) { next.template load_one<i>(loader, loader, wave); });
    }
    at.move((j & 1) ? -2 * kTileBytes : 2 * kTileBytes);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup

  __syncthreads();  // nobody reads the tiles any more
  if (!wave_active) return;
  const float l_tot = lane_pair_sum(l_run);
  const float inv_l = 1.f / l_tot;
  using Out = RowTurn<D, 2>;
  using Rest = RowTurn<D, 1>;
  char* mine = smem + wave * (Out::kBytes + Rest::kBytes);
#pragma unroll
  for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o_acc[db][4 * g + e] * inv_l;
      const u32x2 w = {pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
      Out::put(mine, r, h, db, g, w);
      if (out_rest)
        Rest::put(mine + Out::kBytes, r, h, db, g,
                  pack_rest(o[0] - bf16_lo(w[0]), o[1] - bf16_hi(w[0]), o[2] - bf16_lo(w[1]), o[3] - bf16_hi(w[1])));
    }
  const int64_t row = (int64_t(b) * T + q0) * (int64_t(s.H) * D) + int64_t(head) * D;
  Out::store(mine, reinterpret_cast<char*>(out + row), int64_t(s.H) * D * 2, T - q0, lane);
  if (out_rest) Rest::store(mine + Out::kBytes, reinterpret_cast<char*>(out_rest + row), int64_t(s.H) * D, T - q0, lane);
  // minus the row's log-sum of exponentials, in units of a score: what the backward's S chains start from
  if (h == 0 && q_row < T) neg_lse_out[int64_t(bh) * T + q_row] = -(m_run + __log2f(l_tot)) / c;
}

// ============================================================================ dQ
// S^T = K Q^T - lse / c, P^T = exp2(c S^T), dP^T = V dO^T - delta, dS^T = P^T dP^T, dQ^T += K^T dS^T: the
// row constants are the accumulators' initial values. Also
// delta = rowsum(dO O) for the dK / dV kernels. A tile is two 32-key halves with the same score registers in turn;
// the first half's dQ products are issued under the second one's exponentials.
template <int D, bool kDrop>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 && !kDrop ? 3 : 2))) void window_dq_kernel(
    const bf16_raw* __restrict__ qkv, const bf16_raw* __restrict__ out, const uint8_t* __restrict__ out_rest,
    const bf16_raw* __restrict__ dout, const float* __restrict__ neg_lse_in, float* __restrict__ neg_delta_out,
    bf16_raw* __restrict__ dqkv, Shape s, DropoutParams drop) {
  constexpr int kKSteps = D / 16;
  constexpr int kDBlocks = D / 32;
  constexpr int kTileBytes = kBN * D * 2;
  constexpr int kAhead = D == 128 && kDrop ? 3 : 6;  // fragments in flight (the dropout words take registers)
  extern __shared__ __attribute__((aligned(256))) char smem[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

  TileLoader<D> loader;
  loader.init(tok_stride, wave, lane);
  loader.load(k_base, tiles[0] * kBN, T - 1, smem, wave);
  loader.load(v_base, tiles[0] * kBN, T - 1, smem + kTileBytes, wave);
  auto following = [&](int j) {  // tile j + 1 (behind the last: nothing)
    const bool more = j + 1 < tiles.total;
    const int first = tiles[more ? j + 1 : j] * kBN, last = more ? T - 1 : -1;
    return NextTile<D>{loader.aim(k_base, first, last), loader.aim(v_base, first, last), smem + ((j + 1) & 1) * 2 * kTileBytes};
  };
  bf16x8 qf[kKSteps], dof[kKSteps];
  float dpart = 0.f;
  {
    const int64_t row = (int64_t(b) * T + q_ld) * o_stride + int64_t(head) * D;
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      qf[ks] = *reinterpret_cast<const bf16x8*>(q_base + int64_t(q_ld) * tok_stride + 16 * ks + 8 * h);
      dof[ks] = *reinterpret_cast<const bf16x8*>(dout + row + 16 * ks + 8 * h);
      const bf16x8 of = *reinterpret_cast<const bf16x8*>(out + row + 16 * ks + 8 * h);
      const u32x2 rest = *reinterpret_cast<const u32x2*>(out_rest + row + 16 * ks + 8 * h);
      float lo[8];
      unpack_rest(rest, lo);
#pragma unroll
      for (int j = 0; j < 8; ++j) dpart += (float)dof[ks][j] * ((float)of[j] + lo[j]);
    }
  }
  const float delta = lane_pair_sum(dpart);
  const float neg_lse = neg_lse_in[int64_t(bh) * T + q_ld];
  if (h == 0 && q_row < T) neg_delta_out[int64_t(bh) * T + q_row] = -delta;
  asm volatile("" ::"v"(neg_lse), "v"(delta));  // arrived here, not inside the loop
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) asm volatile("" ::"v"(__builtin_bit_cast(u32x4, qf[ks])));
  const float c = s.scale * kLog2e;
  TileAddrSmall<D> at;
  at.init(lds_addr(smem), lane);

  f32x16 dq_acc[kDBlocks];
#pragma unroll
  for (int i = 0; i < kDBlocks; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) dq_acc[i][j] = 0.f;

  for (int j = 0; j < tiles.total; ++j) {
    const int key0 = tiles[j] * kBN;
    next_tile_ready();
    const NextTile<D> next = following(j);

    auto tile = [&](bool masked) {
      // One stream of products: S and dP of the first half (in turn, n odd is dP), of the second half, then dQ of the
      // first half and of the second. Product n's fragment is requested behind product n - kAhead.
      constexpr int kN = 2 * kKSteps, kTN = 2 * kDBlocks, kAll = 2 * kN + 2 * kTN;
      u32x4 f[kAhead];
      u32x2 tlo[kAhead], thi[kAhead];
      auto request = [&](auto n) {
        if constexpr (n < 2 * kN) {
          constexpr int kb = n / kN, m = n % kN;
          f[n % kAhead] = read16<(m % 2 ? kTileBytes : 0) + kb * 64 * D>(at.row(m / 2));
        } else if constexpr (n < kAll) {
          constexpr int m = n - 2 * kN, k = m / kDBlocks, db = m % kDBlocks;  // 16-key step, column block
          tlo[n % kAhead] = read_tr8<k * 32 * D>(at.tr(db, 0));
          thi[n % kAhead] = read_tr8<k * 32 * D>(at.tr(db, 1));
        }
      };
      static_for<0, kAhead>(request);
      f32x16 s_acc, dp_acc;  // of the half in hand
      bf16x8 ds[4];
      auto start = [&](int kb) {
        float s0 = neg_lse, dp0 = -delta, first[16];
        asm volatile("" : "+v"(s0), "+v"(dp0));  // (16 copies each are made here, not held through the loop)
#pragma unroll
        for (int i = 0; i < 16; ++i) first[i] = s0;
        if (masked) start_masked(s, q_row, key0 + 32 * kb, h, first);  // wave-uniform
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s_acc[i] = first[i];
          dp_acc[i] = dp0;
        }
      };
      auto multiply = [&](auto n) {
        constexpr int last = n + kAhead - 1 < kAll - 1 ? n + kAhead - 1 : kAll - 1;  // newest request
        constexpr int last1 = last < 2 * kN - 1 ? last : 2 * kN - 1;
        constexpr int younger = (last1 > n ? last1 - n : 0) + 2 * (last >= 2 * kN ? last - (n >= 2 * kN ? n : 2 * kN - 1) : 0);
        if constexpr (n < 2 * kN) {
          constexpr int m = n % kN;
          wait_for<younger>(f[n % kAhead]);
          const bf16x8 a = __builtin_bit_cast(bf16x8, f[n % kAhead]);
          if constexpr (m % 2 == 0) s_acc = mfma32(a, qf[m / 2], s_acc);
          else dp_acc = mfma32(a, dof[m / 2], dp_acc);
        } else {
          constexpr int m = n - 2 * kN, k = m / kDBlocks, db = m % kDBlocks;
          wait_for<younger>(tlo[n % kAhead], thi[n % kAhead]);
          dq_acc[db] = mfma32(join(tlo[n % kAhead], thi[n % kAhead]), ds[k], dq_acc[db]);
        }
        request(std::integral_constant<int, n + kAhead>{});
        next.template behind<n>(loader, loader, wave);
        __builtin_amdgcn_sched_barrier(0);
      };
      auto prepare = [&](int kb) {  // dropout, before the elements
        if constexpr (kDrop) {
          uint32_t words[4];
          dropout_words_for_query(drop, bh, q_row, key0 + kb * 32, h, lane, words);
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool keep = ((words[g] >> (8 * e)) & 0xffu) >= drop.threshold;
              const float dp_true = dp_acc[4 * g + e] + delta;
              dp_acc[4 * g + e] = (keep ? dp_true * drop.keep_scale : 0.f) - delta;
            }
        }
      };
      auto element = [&](auto i) {
        constexpr int e = i;
        s_acc[e] = __builtin_amdgcn_exp2f(s_acc[e] * c) * dp_acc[e];
      };
      auto pack_half = [&](auto kb) {
        const f32x16& a = s_acc;
        constexpr int at = 2 * kb;
        ds[at] = pack_acc8(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7]);
        ds[at + 1] = pack_acc8(a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15]);
      };
      start(0);
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, kN>(multiply);
      prepare(0);
      static_for<0, 16>(element);
      pack_half(std::integral_constant<int, 0>{});
      __builtin_amdgcn_sched_barrier(0);
      start(1);
      __builtin_amdgcn_sched_barrier(0);
      static_for<kN, 2 * kN>(multiply);
      prepare(1);
      // the second half's elements under the first half's dQ, from the third product on (the chains take that long)
      static_for<2 * kN, 2 * kN + kTN>([&](auto n) {
        multiply(n);
        constexpr int j = n - 2 * kN;
        if constexpr (j >= 2) static_for<(j - 2) * 16 / (kTN - 2), (j - 1) * 16 / (kTN - 2)>(element);
        __builtin_amdgcn_sched_barrier(0);
      });
      pack_half(std::integral_constant<int, 1>{});
      static_for<2 * kN + kTN, kAll>(multiply);
    };
    if (wave_active && tile_seen(s, key0, q0)) {  // wave-uniform, both
      tile(tile_masked(s, key0, q0));
    } else {
      static_for<0, NextTile<D>::kLoads>([&](auto i) { next.template load_one<i>(loader, loader, wave); });
    }
    at.move((j & 1) ? -2 * kTileBytes : 2 * kTileBytes);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup

  __syncthreads();  // nobody reads the tiles any more
  using Turn = RowTurn<D, 2>;
  char* mine = smem + wave * Turn::kBytes;
#pragma unroll
  for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const u32x2 w = {pack_bf16x2(dq_acc[db][4 * g] * s.scale, dq_acc[db][4 * g + 1] * s.scale),
                       pack_bf16x2(dq_acc[db][4 * g + 2] * s.scale, dq_acc[db][4 * g + 3] * s.scale)};
      Turn::put(mine, r, h, db, g, w);
    }
  bf16_raw* dq_rows = dqkv + (int64_t(b) * T + q0) * tok_stride + int64_t(head) * D;
  Turn::store(mine, reinterpret_cast<char*>(dq_rows), tok_stride * 2, T - q0, lane);
}

}  // namespace

void window_attention_forward(const void* qkv, void* out, void* out_rest, float* neg_lse, int B, int T, int H, int D, int window, int sinks,
                              float softmax_scale, float dropout_p, uint64_t seed, hipStream_t stream) {
  const Shape s{B, T, H, window, sinks, softmax_scale};
  const dim3 grid((unsigned)(ceil_div(T, kBM) * B * H)), block(kThreads);
  const DropoutParams drop = make_dropout_params(dropout_p, seed);
  const size_t lds = size_t(2) * 2 * kBN * D * 2;
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, block, lds, stream, (const bf16_raw*)qkv, (bf16_raw*)out, (uint8_t*)out_rest, neg_lse, s, drop);
  };
  if (D == 64) {
    if (drop.threshold) launch(window_fwd_kernel<64, true>);
    else launch(window_fwd_kernel<64, false>);
  } else {
    if (drop.threshold) launch(window_fwd_kernel<128, true>);
    else launch(window_fwd_kernel<128, false>);
  }
}

void window_attention_dq(const void* qkv, const void* out, const void* out_rest, const void* dout, const float* neg_lse,
                         float* neg_delta, void* dqkv, int B, int T, int H, int D, int window, int sinks, float softmax_scale,
                         float dropout_p, uint64_t seed, hipStream_t stream) {
  const Shape s{B, T, H, window, sinks, softmax_scale};
  const dim3 grid((unsigned)(ceil_div(T, kBM) * B * H)), block(kThreads);
  const DropoutParams drop = make_dropout_params(dropout_p, seed);
  const size_t lds = size_t(2) * 2 * kBN * D * 2;
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, block, lds, stream, (const bf16_raw*)qkv, (const bf16_raw*)out, (const uint8_t*)out_rest,
                       (const bf16_raw*)dout, neg_lse, neg_delta, (bf16_raw*)dqkv, s, drop);
  };
  if (D == 64) {
    if (drop.threshold) launch(window_dq_kernel<64, true>);
    else launch(window_dq_kernel<64, false>);
  } else {
    if (drop.threshold) launch(window_dq_kernel<128, true>);
    else launch(window_dq_kernel<128, false>);
  }
}

}  // namespace pda
