// Shared pieces of the sliding-window attention kernels: which tiles a workgroup visits, tiles loaded to LDS
// directly, and LDS reads by hand (see attention_window.hip).
#pragma once

#include <type_traits>

#include "attention_common.h"
#include "pda_kernels.h"

namespace pda {
namespace window {

using namespace attn;
constexpr int kThreads = 256;
constexpr int kBM = 128;  // rows owned by a workgroup
constexpr int kBN = 64;   // rows per streamed tile

template <int kBegin, int kEnd, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (kBegin < kEnd) {
    f(std::integral_constant<int, kBegin>{});
    static_for<kBegin + 1, kEnd>(f);
  }
}

// ---- LDS reads in flight. An asm output counts as written at once, so nothing may touch it before wait_for (which
// ties the registers to the wait). A kernel that uses these must not spill, its register budget is chosen so, and the
// build checks the compiler's output for both. kYounger: reads requested after the one awaited.
template <int kOff>
__device__ __forceinline__ u32x4 read16(unsigned addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(kOff));
  return v;
}
template <int kOff>
__device__ __forceinline__ u32x2 read_tr8(unsigned addr) {
  u32x2 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(kOff));
  return v;
}
template <int kYounger, typename T>
__device__ __forceinline__ void wait_for(T& v) {
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(v) : "i"(kYounger));
}
template <int kYounger, typename T>
__device__ __forceinline__ void wait_for(T& a, T& b) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(a), "+v"(b) : "i"(kYounger));
}
__device__ __forceinline__ bf16x8 join(u32x2 lo, u32x2 hi) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3));
}

// The XOR that tile_off applies to the 16-byte chunks of a row.
template <int D>
__device__ __forceinline__ int tile_xor(int row) {
  if constexpr (D == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 1) | (((row >> 3) & 1) << 1);
  else return ((row & 3) << 2) | ((row >> 2) & 3);
}

// This lane's addresses in a tile at LDS offset `base`: by rows (row r of a 32-row block, chunk 2 ks + h; block
// kb is kb * 64 D bytes further) and transposed (16-row step k, 32-column block db: as attn::tr_fragment; step k
// is k * 32 D bytes further, the second half of the fragment 8 rows on is an address of its own).
template <int D>
struct TileAddr {
  unsigned row[D / 16], tr[D / 32][2];
  __device__ __forceinline__ void init(unsigned base, int lane) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) row[ks] = base + (unsigned)tile_off<D>(r, 2 * ks + h);
    const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int col = db * 32 + 16 * (g & 1) + 4 * p;
        tr[db][half] = base + (unsigned)(tile_off<D>(4 * (g >> 1) + q + 8 * half, col >> 3) + (col & 7) * 2);
      }
  }
  __device__ __forceinline__ void move(int by) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) row[ks] += by;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) tr[db][0] += by, tr[db][1] += by;
  }
};

// The same addresses out of three registers: steps, column blocks and halves only flip bits inside a row (tiles
// start at multiples of a row), at an instruction per read.
template <int D>
struct TileAddrSmall {
  unsigned row0, tr0, tr1;
  __device__ __forceinline__ void init(unsigned base, int lane) {
    TileAddr<D> at;
    at.init(base, lane);
    row0 = at.row[0], tr0 = at.tr[0][0], tr1 = at.tr[0][1];
  }
  __device__ __forceinline__ unsigned row(int ks) const { return row0 ^ (unsigned)(32 * ks); }
  __device__ __forceinline__ unsigned tr(int db, int half) const { return (half ? tr1 : tr0) ^ (unsigned)(64 * db); }
  __device__ __forceinline__ void move(int by) { row0 += by, tr0 += by, tr1 += by; }
};

// Moves 64-row tiles of [rows][D] bf16 (row pitch in bytes) into LDS, swizzled as tile_off: lane p of a wave's
// load i lands on row 16 wave + i kRows + p / kChunks, slot p % kChunks, and fetches the chunk that belongs there.
// Rows past `last` are out of the source's range: the hardware fills them with zeros.
template <int D>
struct TileLoader {
  static constexpr int kChunks = D / 8, kRows = 64 / kChunks, kLoads = 16 / kRows;
  unsigned pitch;
  unsigned off[kLoads];  // this lane's, for a whole tile
  __device__ __forceinline__ void init(int64_t row_stride, int wave, int lane) {
    pitch = (unsigned)row_stride * 2u;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = 16 * wave + i * kRows + lane / kChunks;
      off[i] = (unsigned)row * pitch + (unsigned)(((lane % kChunks) ^ tile_xor<D>(row)) * 16);
    }
  }
  // rows first .. first + 63 of `base` (a negative `last`: none, all zeros)
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t aim(const bf16_raw* base, int first, int last) const {
    const int left = min(last - first, 63);
    const char* start = reinterpret_cast<const char*>(base) + int64_t(first) * pitch;  // wave-uniform
    return __builtin_amdgcn_make_buffer_rsrc((void*)start, 0, left < 0 ? 0 : (int)((unsigned)left * pitch + 2u * D), 0x00027000);
  }
  template <int I>
  __device__ __forceinline__ void load_one(__amdgpu_buffer_rsrc_t src, char* tile, int wave) const {
    typedef __attribute__((address_space(3))) void lds_ptr_t;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr_t*)(tile + 16 * wave * 2 * D + I * kRows * 2 * D), 16, (int)off[I], 0, 0, 0);
  }
  __device__ __forceinline__ void load(const bf16_raw* base, int first, int last, char* tile, int wave) const {
    const auto src = aim(base, first, last);
    static_for<0, kLoads>([&](auto i) { load_one<i>(src, tile, wave); });
  }
};

// The next tile's two loads (K and V, or Q and dO) of a wave, one at a time between the products: a burst of them
// would keep the wave from issuing products for as long as the loads' addresses take (500 cycles at D = 128).
template <int D>
struct NextTile {
  static constexpr int kLoads = 2 * TileLoader<D>::kLoads;
  __amdgpu_buffer_rsrc_t a, b;
  char* dst;
  template <int I>
  __device__ __forceinline__ void load_one(const TileLoader<D>& la, const TileLoader<D>& lb, int wave) const {
    constexpr int kHalf = TileLoader<D>::kLoads;
    if constexpr (I < kHalf) la.template load_one<I>(a, dst, wave);
    else if constexpr (I < kLoads) lb.template load_one<I - kHalf>(b, dst + kBN * D * 2, wave);
  }
  // behind product n: every other one from the first on
  template <int N>
  __device__ __forceinline__ void behind(const TileLoader<D>& la, const TileLoader<D>& lb, int wave) const {
    if constexpr (N % 2 == 0 && N / 2 < kLoads) load_one<N / 2>(la, lb, wave);
  }
};

// All loads into LDS that this wave has issued have landed; then every wave's have, and every wave is done with
// the tile before.
__device__ __forceinline__ void next_tile_ready() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

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

// A wave's 32 rows of results, turned around in LDS of its own so that they leave in whole rows (from the
// accumulators a store would touch 32 rows with 16 bytes each). The 16-byte chunks of a row are XORed with its index.
template <int D, int kSize>  // kSize: bytes of a value, 2 or 1
struct RowTurn {
  static constexpr int kRow = D * kSize, kChunks = kRow / 16, kBytes = 32 * kRow;
  __device__ __forceinline__ static char* at(char* mem, int row, int chunk) {
    return mem + row * kRow + ((chunk ^ (row & (kChunks - 1))) << 4);
  }
  // columns 32 db + 8 g + 4 h .. +3 of row r
  template <typename V>
  __device__ __forceinline__ static void put(char* mem, int r, int h, int db, int g, V w) {
    static_assert(sizeof(V) == 4 * kSize);
    const int byte = (32 * db + 8 * g) * kSize;
    *reinterpret_cast<V*>(at(mem, r, byte / 16) + byte % 16 + 4 * h * kSize) = w;
  }
  // the first `rows` rows to `to`, `pitch` bytes apart
  __device__ __forceinline__ static void store(const char* mem, char* to, int64_t pitch, int rows, int lane) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes
#pragma unroll
    for (int i = 0; i < kBytes / 1024; ++i) {
      const int row = (64 * i + lane) / kChunks, chunk = (64 * i + lane) % kChunks;
      const u32x4 w = *reinterpret_cast<const u32x4*>(at(const_cast<char*>(mem), row, chunk));
      if (row < rows) *reinterpret_cast<u32x4*>(to + row * pitch + chunk * 16) = w;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before it is written again
  }
};

// Score accumulators of the 32 keys from `key0` on start from minus infinity where the query (on the lane) does
// not see the key: the products leave it there, so the maximum ignores it and its probability is zero.
__device__ __forceinline__ void start_masked(const Shape& s, int q_row, int key0, int h, float (&acc)[16]) {
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (!visible(s, q_row, key0 + acc_row(i, h))) acc[i] = -INFINITY;
    __builtin_amdgcn_sched_barrier(0);  // (few registers: one comparison at a time)
  }
}

}  // namespace window
}  // namespace pda
