// dK and dV of sliding-window attention (attention_window.hip has the rest and the outline).
//
// Registers decide this kernel. A wave keeps K and V of its 32 keys (operands of S and dP) and sums dK and dV; with
// 128 columns that is 64 + 128 registers before the first score, so one wave runs on a SIMD and has to overlap its
// own matrix and vector work: a tile's two sub-tiles are pipelined, exponentials behind matrix instructions. The sums
// belong in the accumulator file, everything the vector unit touches in ordinary registers. The compiler puts either
// all matrix results in the one or all in the other (and then moves some 450 registers per tile between them), so the
// sums' products are inline assembly on accumulator registers.
#include "attention_window.h"

namespace pda {
using attn::DropoutParams;
using attn::make_dropout_params;
namespace {

using namespace window;

// ========================================================================= dK / dV
// S = Q K^T - lse / c, P = exp2(c S), dP = dO V^T - delta, dS = P dP, dV^T += dO^T P, dK^T += Q^T dS. A tile is
// two 32-query sub-tiles, pipelined like the halves of the dQ kernel.
//
// kFar: partial sums of the queries beyond the window, for the first `rows` (sinks rounded up to 32) keys: fp32
// [B * H][chunks][2: dK, dV][rows][D]. A workgroup owns 32 sinks and a chunk of those queries; its waves share the
// keys and split the queries, 32 each of the two tiles in LDS, and their sums meet in LDS.
struct FarSums {
  float* ptr;
  int chunks, tiles_per_chunk, rows;  // tiles_per_chunk is even
};

// acc += a b with acc in accumulator registers. The compiler does not know that this is a matrix instruction: the
// nop covers operands that vector instructions have just written, settle() whatever reads acc after the last one, the
// compiler's own copies included (so a loop that they may leave or enter settles in every trip; the build checks what
// the compiler made of it); products of one acc are at least four apart, and nothing else touches it in between.
__device__ __forceinline__ void mfma32_acc(bf16x8 a, bf16x8 b, f32x16& acc) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void settle(f32x16 (&a)[4], f32x16 (&b)[4]) {
  asm volatile("s_nop 15\n\ts_nop 3" : "+a"(a[0]), "+a"(a[1]), "+a"(a[2]), "+a"(a[3]), "+a"(b[0]), "+a"(b[1]), "+a"(b[2]), "+a"(b[3]));
}

template <int D, bool kDrop, bool kFar>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? (kDrop || kFar ? 2 : 3) : 1))) void window_dkv_kernel(
    const bf16_raw* __restrict__ qkv, const bf16_raw* __restrict__ dout, const float* __restrict__ neg_lse,
    const float* __restrict__ neg_delta, bf16_raw* __restrict__ dqkv, FarSums far, Shape s, DropoutParams drop) {
  constexpr int kKSteps = D / 16;
  constexpr int kDBlocks = D / 32;
  constexpr int kTileBytes = kBN * D * 2;
  constexpr int kAhead = D == 64 ? 3 : 6;  // fragments in flight
  // [2][Q tile | dO tile], then [2][64 x (-lse / c) | 64 x (-delta)] fp32 row constants
  extern __shared__ __attribute__((aligned(256))) char smem[];
  char* row_smem = smem + 4 * kTileBytes;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;

  const int BH = s.B * s.H, T = s.T;
  const int bh = blockIdx.x % BH;
  const int n_blocks = far.rows / 32;  // of sinks
  const int kt = kFar ? (blockIdx.x / BH) % n_blocks : blockIdx.x / BH;
  const int chunk = kFar ? blockIdx.x / (BH * n_blocks) : 0;
  const int b = bh / s.H, head = bh % s.H;
  const int64_t tok_stride = int64_t(3) * s.H * D, o_stride = int64_t(s.H) * D;
  const bf16_raw* q_base = qkv + int64_t(b) * T * tok_stride + int64_t(head) * D;
  const bf16_raw* k_base = q_base + int64_t(s.H) * D;
  const bf16_raw* v_base = q_base + int64_t(2) * s.H * D;
  const bf16_raw* do_base = dout + int64_t(b) * T * o_stride + int64_t(head) * D;
  const float* lse_row = neg_lse + int64_t(bh) * T;
  const float* delta_row = neg_delta + int64_t(bh) * T;

  const int key0 = kFar ? kt * 32 : kt * kBM + wave * 32;  // first key of this wave
  const int key = key0 + r;                                // this lane's key
  const int key_ld = key < T ? key : T - 1;

  // Query tiles: the window's (from the diagonal to the last query that sees the last key), or this chunk's
  // share of those beyond it.
  const int n_tiles = (T + kBN - 1) / kBN;
  int first_tile, end_tile;
  if (kFar) {
    first_tile = (kt * 32 + s.window) / kBN + chunk * far.tiles_per_chunk;
    end_tile = min(n_tiles, first_tile + far.tiles_per_chunk);
  } else {
    first_tile = kt * kBM / kBN;
    const int last_q = min(T - 1, kt * kBM + kBM - 1 + s.window - 1);
    end_tile = last_q / kBN + 1;
  }
  // This lane's key belongs to the queries q_lo <= q < q_hi of this workgroup (none for a key past the end).
  const int q_lo = kFar ? key + s.window : key;
  const int q_hi = kFar ? (key < s.sinks ? min(T, end_tile * kBN) : 0) : min(key + s.window, T);
  // Are some (query, key) pairs of this wave's 32 keys and the 32 queries from qs masked? (wave-uniform)
  auto edge = [&](int qs) {
    return kFar ? qs < key0 + 31 + s.window || qs + 31 >= min(T, end_tile * kBN) || key0 + 32 > s.sinks
                : qs < key0 + 31 || qs + 31 >= min(key0 + s.window, T);
  };

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

  TileLoader<D> q_loader, do_loader;
  q_loader.init(tok_stride, wave, lane);
  do_loader.init(o_stride, wave, lane);
  auto fetch_constants = [&](int tile, int buf) {
    typedef __attribute__((address_space(1))) const void global_ptr_t;
    typedef __attribute__((address_space(3))) void lds_ptr_t;
    if (wave < 2) {  // wave 0: -lse / c, wave 1: -delta of the tile's 64 queries
      const float* src = (wave == 0 ? lse_row : delta_row) + min(tile * kBN + lane, T - 1);
      __builtin_amdgcn_global_load_lds((global_ptr_t*)src, (lds_ptr_t*)(row_smem + buf * 512 + wave * 256), 4, 0, 0);
    }
  };
  auto fetch = [&](int tile, int buf) {
    char* dst = smem + buf * 2 * kTileBytes;
    q_loader.load(q_base, tile * kBN, T - 1, dst, wave);
    do_loader.load(do_base, tile * kBN, T - 1, dst + kTileBytes, wave);
    fetch_constants(tile, buf);
  };
  [[maybe_unused]] NextTile<D> following;  // what the stream of both sub-tiles loads on its way
  if constexpr (!kFar) fetch(first_tile, 0);
  bf16x8 kf[kKSteps], vf[kKSteps];
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) {
    kf[ks] = *reinterpret_cast<const bf16x8*>(k_base + int64_t(key_ld) * tok_stride + 16 * ks + 8 * h);
    vf[ks] = *reinterpret_cast<const bf16x8*>(v_base + int64_t(key_ld) * tok_stride + 16 * ks + 8 * h);
  }
  // K and V arrive here, beside the first tile, not at their first use inside the loop
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) {
    asm volatile("" ::"v"(__builtin_bit_cast(u32x4, kf[ks])));
    asm volatile("" ::"v"(__builtin_bit_cast(u32x4, vf[ks])));
  }
  TileAddrSmall<D> at;
  at.init(lds_addr(smem), lane);
  unsigned row_at = lds_addr(row_smem) + 16u * (unsigned)h;  // row constants 4 h ..; 8 rows further: + 32 bytes

  // The products of a tile are one stream: S and dP of sub-tile 0 (in turn: two chains, so that neither waits for
  // itself), of sub-tile 1, then dV and dK of sub-tile 0 and of 1. Product n's fragment is requested behind product
  // n - kAhead; fragments of the first two parts are one LDS read, transposed ones two.
  constexpr int kN = 2 * kKSteps;   // S and dP products of a sub-tile: n / 2 is the step, n odd is dP
  constexpr int kTN = 4 * kDBlocks; // dV and dK: n / 2 / kDBlocks is the 16-query step, n / 2 % kDBlocks the column block, n odd is dK
  f32x16 s_acc[2], dp_acc[2];
  [[maybe_unused]] float delta_c[2][kDrop ? 16 : 1];
  u32x4 f[kAhead], ca[4], cd[4];
  u32x2 tlo[kAhead], thi[kAhead];
  // kSubs: sub-tiles in the stream (2, or the one at offset 0)
  auto request = [&](auto subs, auto n) {
    constexpr int kChain = subs * kN;
    if constexpr (n < kChain) {
      constexpr int sub = n / kN, m = n % kN;
      f[n % kAhead] = read16<(m % 2 ? kTileBytes : 0) + sub * 64 * D>(at.row(m / 2));
    } else if constexpr (n < kChain + subs * kTN) {
      constexpr int sub = (n - kChain) / kTN, m = (n - kChain) % kTN, k = 2 * sub + m / (2 * kDBlocks), db = m / 2 % kDBlocks;
      tlo[n % kAhead] = read_tr8<(m % 2 ? 0 : kTileBytes) + k * 32 * D>(at.tr(db, 0));
      thi[n % kAhead] = read_tr8<(m % 2 ? 0 : kTileBytes) + k * 32 * D>(at.tr(db, 1));
    }
  };
  // Row constants of a sub-tile: 8 reads, requested ahead like a fragment.
  auto request_constants = [&](auto sub) {
    static_for<0, 4>([&](auto g) {
      ca[g] = read16<sub * 128 + g * 32>(row_at);
      cd[g] = read16<256 + sub * 128 + g * 32>(row_at);
    });
  };
  // The accumulators of sub-tile `sub` (32 queries from qs) start from its row constants, masked pairs from minus
  // infinity: their probabilities come out as zero, and everything behind is one straight line of code.
  auto start = [&](auto sub, int qs) {
    asm volatile("" : "+v"(ca[0]), "+v"(ca[1]), "+v"(ca[2]), "+v"(ca[3]));
    asm volatile("" : "+v"(cd[0]), "+v"(cd[1]), "+v"(cd[2]), "+v"(cd[3]));
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s_acc[sub][4 * g + e] = __uint_as_float(ca[g][e]);
        dp_acc[sub][4 * g + e] = __uint_as_float(cd[g][e]);
        if constexpr (kDrop) delta_c[sub][4 * g + e] = __uint_as_float(cd[g][e]);
      }
    if (edge(qs)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int q = qs + acc_row(i, h);
        if (q < q_lo || q >= q_hi) s_acc[sub][i] = -INFINITY;
      }
    }
  };
  uint32_t keep_mask[2] = {0xffffu, 0xffffu};
  auto element = [&](auto sub, int i) {
    const float p = __builtin_amdgcn_exp2f(s_acc[sub][i] * c);
    if constexpr (kDrop) {
      const bool keep = (keep_mask[sub] >> i) & 1;
      const float nd = delta_c[sub][i];
      const float dp = (keep ? (dp_acc[sub][i] - nd) * drop.keep_scale : 0.f) + nd;
      dp_acc[sub][i] = p * dp;
      s_acc[sub][i] = keep ? p * drop.keep_scale : 0.f;
    } else {
      s_acc[sub][i] = p;
      dp_acc[sub][i] = p * dp_acc[sub][i];
    }
  };
  auto pack = [&](const f32x16& v, int o) {
    return pack_acc8(v[o], v[o + 1], v[o + 2], v[o + 3], v[o + 4], v[o + 5], v[o + 6], v[o + 7]);
  };
  bf16x8 pp[2], pds[2];  // P and dS of the sub-tile whose dV and dK products run
  auto pack_sub = [&](auto sub) {
    pp[0] = pack(s_acc[sub], 0), pp[1] = pack(s_acc[sub], 8);
    pds[0] = pack(dp_acc[sub], 0), pds[1] = pack(dp_acc[sub], 8);
  };
  // Reads requested behind that of product n when product n is due.
  auto multiply = [&](auto subs, auto n) {
    constexpr int kChain = subs * kN, kAll = kChain + subs * kTN;
    constexpr int last = n + kAhead - 1 < kAll - 1 ? n + kAhead - 1 : kAll - 1;  // newest request
    constexpr int singles = (last < kChain - 1 ? last : kChain - 1) > n ? (last < kChain - 1 ? last : kChain - 1) - n : 0;
    constexpr int pairs = last >= kChain ? last - (n >= kChain ? n : kChain - 1) : 0;
    constexpr int consts = subs == 2 && n > kN - kAhead && n < kN ? 8 : 0;  // requested behind product kN - kAhead
    constexpr int younger = singles + 2 * pairs + consts < 15 ? singles + 2 * pairs + consts : 15;
    if constexpr (n < kChain) {
      constexpr int sub = n / kN, m = n % kN;
      wait_for<younger>(f[n % kAhead]);
      const bf16x8 a = __builtin_bit_cast(bf16x8, f[n % kAhead]);
      if constexpr (m % 2 == 0) s_acc[sub] = mfma32(a, kf[m / 2], s_acc[sub]);
      else dp_acc[sub] = mfma32(a, vf[m / 2], dp_acc[sub]);
    } else {
      constexpr int m = (n - kChain) % kTN, k = m / (2 * kDBlocks), db = m / 2 % kDBlocks;
      wait_for<younger>(tlo[n % kAhead], thi[n % kAhead]);
      const bf16x8 a = join(tlo[n % kAhead], thi[n % kAhead]);
      f32x16& acc = m % 2 ? dk_acc[db] : dv_acc[db];
      const bf16x8& b = m % 2 ? pds[k] : pp[k];
      if constexpr (D == 128) mfma32_acc(a, b, acc);
      else acc = mfma32(a, b, acc);
    }
    if constexpr (subs == 2 && n == kN - kAhead) request_constants(std::integral_constant<int, 1>{});
    request(subs, std::integral_constant<int, n + kAhead>{});
    if constexpr (subs == 2) following.template behind<n>(q_loader, do_loader, wave);
  };
  constexpr std::integral_constant<int, 0> s0{};
  constexpr std::integral_constant<int, 1> s1{};
  // Elements of a sub-tile under `of` products: from the third on (the chains' results take that long).
  auto elements_under = [&](auto sub, auto j, auto of) {
    if constexpr (j >= 2) static_for<(j - 2) * 16 / (of - 2), (j - 1) * 16 / (of - 2)>([&](auto i) { element(sub, i); });
  };
  auto both = [&](int q0) {  // the tile's two sub-tiles, pipelined (no dropout)
    constexpr std::integral_constant<int, 2> subs{};
    constexpr std::integral_constant<int, kN> of_n{};
    constexpr std::integral_constant<int, kTN> of_tn{};
    request_constants(s0);
    static_for<0, kAhead>([&](auto n) { request(subs, n); });
    asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(kAhead));
    start(s0, q0);
    static_for<0, kN>([&](auto n) {
      multiply(subs, n);
      __builtin_amdgcn_sched_barrier(0);
    });
    asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(kAhead));  // the constants are older than the fragments in flight
    start(s1, q0 + 32);
    static_for<kN, 2 * kN>([&](auto n) {
      multiply(subs, n);
      elements_under(s0, std::integral_constant<int, n - kN>{}, of_n);
      __builtin_amdgcn_sched_barrier(0);
    });
    pack_sub(s0);
    static_for<2 * kN, 2 * kN + kTN>([&](auto n) {
      multiply(subs, n);
      elements_under(s1, std::integral_constant<int, n - 2 * kN>{}, of_tn);
      __builtin_amdgcn_sched_barrier(0);
    });
    pack_sub(s1);
    static_for<2 * kN + kTN, 2 * kN + 2 * kTN>([&](auto n) {
      multiply(subs, n);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto one = [&](int qs) {  // the sub-tile at the lane's addresses
    constexpr std::integral_constant<int, 1> subs{};
    request_constants(s0);
    static_for<0, kAhead>([&](auto n) { request(subs, n); });
    asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(kAhead));
    start(s0, qs);
    static_for<0, kN>([&](auto n) {
      multiply(subs, n);
      __builtin_amdgcn_sched_barrier(0);
    });
    if (kDrop) keep_mask[0] = dropout_keep_mask_for_key(drop, bh, qs, h, key, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) element(s0, i);
    pack_sub(s0);
    static_for<kN, kN + kTN>([&](auto n) {
      multiply(subs, n);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  if constexpr (kFar) {
    // two tiles at a time (the second may repeat the first, masked); wave w takes sub-tile w & 1 of tile w >> 1
    at.move((wave >> 1) * 2 * kTileBytes + (wave & 1) * 64 * D);
    row_at += (unsigned)((wave >> 1) * 512 + (wave & 1) * 128);
    for (int j = first_tile; j < end_tile; j += 2) {
      fetch(j, 0);
      fetch(min(j + 1, end_tile - 1), 1);
      next_tile_ready();
      one((j + (wave >> 1)) * kBN + 32 * (wave & 1));
      if constexpr (D == 128) settle(dk_acc, dv_acc);
      __syncthreads();  // everyone has read the two tiles
    }
    // sum over the waves: 2, 3 -> 0, 1, then 1 -> 0 (each through its own place in LDS: 64 lanes x 16 floats a block)
    float* red = reinterpret_cast<float*>(smem);
    auto give = [&](int slot) {
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          red[((slot * 2 * kDBlocks + 2 * db) * 16 + i) * 64 + lane] = dk_acc[db][i];
          red[((slot * 2 * kDBlocks + 2 * db + 1) * 16 + i) * 64 + lane] = dv_acc[db][i];
        }
    };
    auto take = [&](int slot) {
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          dk_acc[db][i] += red[((slot * 2 * kDBlocks + 2 * db) * 16 + i) * 64 + lane];
          dv_acc[db][i] += red[((slot * 2 * kDBlocks + 2 * db + 1) * 16 + i) * 64 + lane];
        }
    };
    if (wave >= 2) give(wave - 2);
    __syncthreads();
    if (wave < 2) take(wave);
    __syncthreads();
    if (wave == 1) give(0);
    __syncthreads();
    if (wave != 0) return;
    take(0);
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

  for (int j = first_tile; j < end_tile; ++j) {
    const int buf = (j - first_tile) & 1;
    next_tile_ready();
    if constexpr (kDrop || D == 64) {
      if (j + 1 < end_tile) fetch(j + 1, buf ^ 1);
    } else {
      const bool more = j + 1 < end_tile;
      const int first = (more ? j + 1 : j) * kBN, last = more ? T - 1 : -1;
      if (more) fetch_constants(j + 1, buf ^ 1);
      following = NextTile<D>{q_loader.aim(q_base, first, last), do_loader.aim(do_base, first, last), smem + (buf ^ 1) * 2 * kTileBytes};
    }
    const int q0 = j * kBN;
    const int next = buf ? -2 * kTileBytes : 2 * kTileBytes;
    // With dropout the pipelined form has no registers left for the masks; with 64 columns three waves on a SIMD, a
    // sub-tile at a time, beat two that pipeline (8 x 1024, 20 heads, window 256: 48 us against 53).
    if constexpr (kDrop || D == 64) {
      one(q0);
      at.move(64 * D);
      row_at += 128;
      one(q0 + 32);
      at.move(next - 64 * D);
      row_at += (buf ? -512 : 512) - 128;
    } else {
      both(q0);
      at.move(next);
      row_at += buf ? -512 : 512;
    }
  }

  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup
  if constexpr (D == 128) settle(dk_acc, dv_acc);
  __syncthreads();  // nobody reads the tiles any more
  using Turn = RowTurn<D, 2>;
  char* mine = smem + wave * Turn::kBytes;
  bf16_raw* dk_rows = dqkv + (int64_t(b) * T + key0) * tok_stride + int64_t(s.H) * D + int64_t(head) * D;
  auto give = [&](const f32x16 (&acc)[kDBlocks], float factor, bf16_raw* rows) {
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x2 w = {pack_bf16x2(acc[db][4 * g] * factor, acc[db][4 * g + 1] * factor),
                         pack_bf16x2(acc[db][4 * g + 2] * factor, acc[db][4 * g + 3] * factor)};
        Turn::put(mine, r, h, db, g, w);
      }
    Turn::store(mine, reinterpret_cast<char*>(rows), tok_stride * 2, T - key0, lane);
  };
  give(dk_acc, s.scale, dk_rows);
  give(dv_acc, 1.f, dk_rows + int64_t(s.H) * D);
}

// The far part's chunks: enough workgroups for two per compute unit, at least eight query tiles each (a chunk
// costs its sinks' owner a pass over its sums).
FarSums far_plan(int B, int T, int H, int window, int sinks) {
  FarSums f{nullptr, 0, 0, 0};
  if (sinks <= 0 || window >= T) return f;
  const int last_sink = sinks < T ? sinks : T;
  f.rows = (last_sink + 31) / 32 * 32;
  const int tiles = (T + kBN - 1) / kBN - window / kBN;  // from the first query beyond the window
  const int64_t owners = int64_t(B) * H * (f.rows / 32);
  int chunks = (int)((512 + owners - 1) / owners);
  const int most = (tiles + 7) / 8;
  if (chunks > most) chunks = most;
  f.tiles_per_chunk = ((tiles + chunks - 1) / chunks + 1) / 2 * 2;
  f.chunks = (tiles + f.tiles_per_chunk - 1) / f.tiles_per_chunk;
  return f;
}

}  // namespace

size_t window_attention_backward_workspace_bytes(int B, int T, int H, int D, int window, int sinks) {
  const FarSums f = far_plan(B, T, H, window, sinks);
  return size_t(B) * H * f.chunks * 2 * f.rows * D * sizeof(float);
}

void window_attention_dkv(const void* qkv, const void* dout, const float* neg_lse, const float* neg_delta, void* dqkv,
                          void* workspace, int B, int T, int H, int D, int window, int sinks, float softmax_scale, float dropout_p,
                          uint64_t seed, hipStream_t stream) {
  const Shape s{B, T, H, window, sinks, softmax_scale};
  FarSums far = far_plan(B, T, H, window, sinks);
  far.ptr = (float*)workspace;
  const dim3 grid((unsigned)(ceil_div(T, kBM) * B * H)), block(kThreads);
  const dim3 far_grid((unsigned)(int64_t(far.rows / 32) * far.chunks * B * H));
  const DropoutParams drop = make_dropout_params(dropout_p, seed);
  const size_t lds = size_t(2) * 2 * kBN * D * 2 + 1024;
  auto launch = [&](auto far_kern, auto kern) {
    if (far.chunks > 0)
      hipLaunchKernelGGL(far_kern, far_grid, block, lds, stream, (const bf16_raw*)qkv, (const bf16_raw*)dout, neg_lse, neg_delta,
                         (bf16_raw*)dqkv, far, s, drop);
    hipLaunchKernelGGL(kern, grid, block, lds, stream, (const bf16_raw*)qkv, (const bf16_raw*)dout, neg_lse, neg_delta,
                       (bf16_raw*)dqkv, far, s, drop);
  };
  if (D == 64) {
    if (drop.threshold) launch(window_dkv_kernel<64, true, true>, window_dkv_kernel<64, true, false>);
    else launch(window_dkv_kernel<64, false, true>, window_dkv_kernel<64, false, false>);
  } else {
    if (drop.threshold) launch(window_dkv_kernel<128, true, true>, window_dkv_kernel<128, true, false>);
    else launch(window_dkv_kernel<128, false, true>, window_dkv_kernel<128, false, false>);
  }
}

}  // namespace pda
