// Pieces shared by the attention kernels: element types, matrix instructions,
// LDS tiles and the lookup of a packed list.
//
// Matrix instructions (64 lanes, l = lane % 32, h = lane / 32): the 32x32x16
// product takes 8 values of A per lane (row l, columns 8h..8h+7) and 8 of B
// (column l, rows 8h..8h+7); its result has column l and rows
// 8 (i / 4) + 4 h + i % 4 in registers i = 0..15.  The kernels choose the
// operands so that what one product leaves is what the next one takes: scores
// come out with a query (or a key) per lane, and 8 consecutive registers of
// them are the B operand of the product that follows, whose A operand reads
// its rows in the same order (4 h + 0..3, then 8 + 4 h + 0..3 of each 16).
// Probabilities never pass through LDS.
#pragma once

#include "mx_common.h"

namespace mx {
namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
struct Elem;

template <>
struct Elem<__bf16> {
  using x8 = bf16x8;
  static constexpr bool kNarrow = false;  // the range of fp32
  static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Elem<_Float16> {
  using x8 = f16x8;
  static constexpr bool kNarrow = true;  // up to 65504
  static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// 2^x by the hardware's instruction: 0 for -inf and for results below the
// normal range.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The other half-wave's value (lane +- 32).
__device__ __forceinline__ float other_half(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(lane_id() < 32 ? r[1] : r[0]);
}

// The smaller, and a row count left of at most `most`.
__device__ __forceinline__ int min_of(int a, int b) { return a < b ? a : b; }
__device__ __forceinline__ int rows_left(int len, int from, int most) {
  const int n = len - from;
  return n < 0 ? 0 : min_of(n, most);
}

// A buffer descriptor of `bytes` bytes from a wave-uniform base: loads past
// them return zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  // In scalar registers whatever the compiler knows of the values: it would
  // loop over the lanes' descriptors otherwise.
  const uint64_t u = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u >> 32));
  void* p = reinterpret_cast<void*>((static_cast<uint64_t>(hi) << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}

// v, of which the compiler knows nothing: what is computed from it in a loop
// stays there instead of taking registers through the loop.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
  asm("" : "+v"(v));
  return v;
}

// The lane's number, counted anew where it is needed.
__device__ __forceinline__ uint32_t lane_again() {
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, opaque(0)));
}

// An offset no descriptor of ours covers (also after a tile's steps).
constexpr uint32_t kOutside = 0x80000000u;

// Bytes of `rows` rows of `width` bytes at a stride, for a descriptor.
__device__ __forceinline__ uint32_t span_bytes(int rows, uint32_t stride, uint32_t width) {
  return rows > 0 ? static_cast<uint32_t>(rows - 1) * stride + width : 0u;
}

// 16 (4) bytes per lane from global memory straight into LDS, at `to` + 16 (4)
// times the lane.
__device__ __forceinline__ void load16_to_lds(__amdgpu_buffer_rsrc_t r, char* to, uint32_t off) {
  auto* dst = (__attribute__((address_space(3))) void*)(to);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, dst, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void load4_to_lds(__amdgpu_buffer_rsrc_t r, char* to, uint32_t off) {
  auto* dst = (__attribute__((address_space(3))) void*)(to);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, dst, 4, off, 0, 0, 0);
}

// A tile of ROWS x DP 16-bit values in LDS: rows of C = DP / 8 chunks of 16
// bytes, chunk c of row r at place c ^ f(r).  LDS serves 256 bytes over 64 banks
// at a time: 16 lanes of a row read (lane l: chunk c of row l) and 32 of a
// transposing read (4 rows x 4 chunks).  f makes both meet every bank once.
template <int DP>
struct Tile {
  static constexpr int C = DP / 8;
  static constexpr int kRow = DP * 2;  // bytes

  static __device__ __forceinline__ int f(int r) {
    if constexpr (C == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (C == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;  // 4 and 12: rows 0..3 fall into different quarters anyway
  }

  // Byte offset of chunk c of row r.
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ f(r)) << 4); }

  // The offset of chunk c + 2 x, and of chunk c + 4 d, of the same row from that
  // of chunk c (c < 2, c < 4): one instruction, no register kept per x or d.
  static __device__ __forceinline__ uint32_t step2(uint32_t at_c, int x) {
    return C == 12 ? (at_c ^ ((x & 1) << 5)) + (x >> 1) * 64 : at_c ^ (x << 5);
  }
  static __device__ __forceinline__ uint32_t step4(uint32_t at_c, int d) {
    return C == 12 ? at_c + d * 64 : at_c ^ (d << 6);
  }

  // The same chunk 8 rows on (from a row r with r & 8 == 0).
  static __device__ __forceinline__ uint32_t next8(uint32_t at_c) {
    return (at_c ^ 32) + 8 * kRow;
  }

  // Copies a tile of ROWS rows from global memory into LDS, without passing
  // through registers: THREADS threads, 16 bytes per lane and instruction, the
  // LDS side contiguous, the global side permuted.  Rows past the descriptor
  // and chunks past `d_chunks` become zeros.
  template <int ROWS, int THREADS>
  struct Loader {
    static constexpr int kAll = ROWS * C;  // 16-byte places
    static constexpr int kPer = kAll / THREADS;
    static_assert(kAll % THREADS == 0, "whole instructions");
    // With a power of two of chunks, an instruction's rows follow the last
    // one's by a fixed number and f repeats: one offset serves all.
    static constexpr bool kOne = THREADS % (16 * C) == 0;
    uint32_t off[kOne ? 1 : kPer];
    uint32_t step;

    __device__ __forceinline__ void init(int tid, uint32_t stride, int d_chunks) {
      step = stride * (THREADS / C);
#pragma unroll
      for (int i = 0; i < (kOne ? 1 : kPer); ++i) {
        const int u = i * THREADS + tid;
        const int r = u / C, c = (u % C) ^ f(r);
        off[i] = c < d_chunks ? static_cast<uint32_t>(r) * stride + c * 16 : kOutside;
      }
    }

    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, char* lds, int wave) const {
      uint32_t o = off[0];
      if constexpr (kOne && kPer > 1) o = opaque(o);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        load16_to_lds(r, lds + (i * THREADS + wave * 64) * 16, kOne ? o + i * step : off[kOne ? 0 : i]);
    }
  };
};

// A lane's places in a tile, from row r0 (a multiple of 16) on: its row's first
// chunk, and its piece of the transposing reads of rows 0..7 of each 16 (8
// columns of the 32 of a block).
template <int DP>
struct Places {
  uint32_t row, tr;
  __device__ __forceinline__ Places(int lane, int r0) {
    using Ti = Tile<DP>;
    const int t = lane & 15, h = lane >> 5;
    const int r = 4 * h + (t >> 2), c = 2 * ((lane >> 4) & 1) + ((t & 3) >> 1);
    row = r0 * Ti::kRow + Ti::at(lane & 31, h);
    tr = r0 * Ti::kRow + Ti::at(r, c) + (t & 1) * 8;
  }
};

template <typename X8>
__device__ __forceinline__ X8 lds_read16(const char* p) {
  return *reinterpret_cast<const X8*>(p);
}

// Transposing LDS read: of each 16 lanes, lane t points at 4 values of row
// t / 4 (columns 4 (t % 4)...); it receives column t of the 4 rows.
__device__ __forceinline__ s16x4 lds_read_tr(const char* p) {
  auto* q = (__attribute__((address_space(3))) s16x4*)(p);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(q);
}

template <typename X8>
__device__ __forceinline__ X8 join(s16x4 a, s16x4 b) {
  return __builtin_bit_cast(X8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A barrier before which all but the wave's last N loads have landed and its LDS
// reads are done (a block barrier of the language would wait for every load).
template <int N>
__device__ __forceinline__ void wait_and_barrier() {
  static_assert(N < 64, "what the counter holds");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------------------
// Packed lists
// ---------------------------------------------------------------------------
// Rows 0..N-1 are cut by B + 1 offsets.  Two more lists without partners hold
// the rows before the first and after the last offset (if there are any), so
// that every row belongs to one list: list 0 those before, lists 1..B the
// caller's, list B + 1 those after.  A launch needs the tiles of BM rows of every
// list without a host copy of the offsets.  With s / BM = a, s % BM = r for a
// list's start and a', r' for its end, it has a' - a tiles and one more if
// r' > r.  So turns 0 .. N / BM - 1 are tiles that exist, turn t in the list
// with a <= t < a' (found by a search), and N / BM + i is list i's one more,
// or nothing.  Blocks without work come last: among the others they would idle
// the dispatcher, which hands the shader engines blocks in turn (256 lists of
// 128 rows with every other block empty: 90 us instead of 60).

struct Span {
  int32_t start;
  int32_t len;  // >= 0
};

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(v >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

template <typename I>
__device__ __forceinline__ int32_t list_start(const I* offsets, int32_t B, int32_t N, int32_t i) {
  if (i <= 0) return 0;
  if (i > B + 1) return N;
  const I o = offsets[i - 1];
  return o < 0 ? 0 : (o > N ? N : static_cast<int32_t>(o));  // malformed offsets stay in bounds
}

// A block's tile: its list's rows and their partners' (queries' keys or keys'
// queries), and its number in the list.
struct Found {
  Span own, other;
  int32_t tile;
};

// Turns rotated within groups of 8, each group by one more than the last: lists
// of a power of two of tiles would give one XCD, or one shader engine, the same
// tile of every list, the longest or the shortest, as blocks go to both in turn.
__device__ __forceinline__ int32_t rotated(int32_t turn, int32_t n) {
  return turn < (n & ~7) ? (turn & ~7) | ((turn + (turn >> 3)) & 7) : turn;
}

// The tile of turn `turn`; false if there is none.  The one more tile is the
// list's first (FIRST: queries, whose first tiles see the fewest keys) or last
// (keys, whose last tiles meet the fewest queries).  Steps of 64 probes narrow the lists down to 63,
// whose bounds on both sides one more load per lane brings (up to 61 lists cost
// one trip to memory, up to 4,030 two: every block waits for them).
template <bool FIRST, typename I>
__device__ __forceinline__ bool find_list(const I* own, const I* other, int32_t B, int32_t N,
                                          int32_t Nother, int bm_shift, int32_t turn, Found* f) {
  const int whole = N >> bm_shift;
  int lo = rotated(turn - whole, B + 2), n = 2;  // one more: the list is known
  if (turn < whole) {
    // Backwards where first tiles are short (the causal mask): long ones first.
    turn = rotated(turn, whole);
    if (FIRST) turn = whole - 1 - turn;
    lo = 0, n = B + 2;
    while (n > 63) {
      const int step = (n + 63) >> 6;
      const int i = lo + lane_id() * step;
      const bool in = i < lo + n && (list_start(own, B, N, i) >> bm_shift) <= turn;
      const int c = __popcll(__ballot(in));  // the first lane's is always at most `turn`
      const int at = (c > 0 ? c - 1 : 0) * step;
      lo += at;
      n = n - at < step ? n - at : step;
    }
  }
  const int i = lo + lane_id();
  const int s = list_start(own, B, N, i), o = list_start(other, B, Nother, i);
  // The last list that starts at or before the turn (those before it with the
  // same start have no whole tile).
  const int c = turn < whole ? __popcll(__ballot(lane_id() < n && (s >> bm_shift) <= turn)) : 1;
  const int at = c > 0 ? c - 1 : 0;  // at most 62
  const int s0 = readlane_i32(s, at), s1 = readlane_i32(s, at + 1);
  const int o0 = readlane_i32(o, at), o1 = readlane_i32(o, at + 1);
  const int list = lo + at, mask = (1 << bm_shift) - 1;
  const bool more = s1 > s0 && (s1 & mask) > (s0 & mask);
  if (turn >= whole && !more) return false;
  f->own = {s0, s1 > s0 ? s1 - s0 : 0};
  f->other = {o0, list > 0 && list <= B && o1 > o0 ? o1 - o0 : 0};
  if (turn >= whole) f->tile = FIRST ? 0 : (s1 >> bm_shift) - (s0 >> bm_shift);
  else f->tile = turn - (s0 >> bm_shift) + (FIRST && more ? 1 : 0);
  return true;
}

// Sum over the lanes up to and including this one.
__device__ __forceinline__ int wave_prefix(int v) {
  // row_shr 1, 2, 4, 8 within 16 lanes, then each row's last to the next rows.
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// The same by rank, for up to 62 lists: tiles with more work come first, across
// all lists (a block's time is its tile's length: the longest must not start
// last).  A lane holds a list; under the causal mask tile t of n has work
// t + 1 + c (QUERIES, c the keys before its queries in tiles) or n - t (keys:
// the queries from its first one on), else every tile of a list has its
// partners' number.  With F(w) the tiles of work w or more, rank r has the
// largest w with F(w) > r and is number r - F(w + 1) of that work in the order
// of the lists.  False if there are no more tiles.
template <bool QUERIES, typename I>
__device__ __forceinline__ bool find_ranked(const I* own, const I* other, int32_t B, int32_t N,
                                            int32_t Nother, int bm_shift, bool causal, int32_t rank,
                                            Found* f) {
  const int i = lane_id();
  const int s = list_start(own, B, N, i), os = list_start(other, B, Nother, i);
  const int e = list_start(own, B, N, i + 1), oe = list_start(other, B, Nother, i + 1);
  const int len = e > s ? e - s : 0;  // past the last list: N to N
  const int olen = i > 0 && i <= B && oe > os ? oe - os : 0;
  const int n = (len + (1 << bm_shift) - 1) >> bm_shift;
  const int top = !causal ? 1 + (olen >> bm_shift)  // the most work of a tile of the list
                  : n + (QUERIES && olen > len ? (olen - len) >> bm_shift : 0);
  auto count = [&](int w) {  // tiles of this list with work w or more
    if (!causal) return top >= w ? n : 0;
    const int k = top - w + 1;
    return k < 0 ? 0 : (k < n ? k : n);
  };
  auto total = [&](int w) { return readlane_i32(wave_prefix(count(w)), 63); };
  if (rank >= total(0)) return false;
  int lo = 0, hi = 1;  // F(lo) > rank >= F(hi)
  while (total(hi) > rank) {
    lo = hi;
    hi *= 2;
  }
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (total(mid) > rank) lo = mid;
    else hi = mid;
  }
  // Of work lo: this list's tiles, and those of the lists before it.
  const int here = count(lo) - count(lo + 1);
  const int k = rank - total(lo + 1) - (wave_prefix(here) - here);
  const int at = __builtin_ctzll(__ballot(k >= 0 && k < here) | (1ull << 63));
  f->own = {readlane_i32(s, at), readlane_i32(len, at)};
  f->other = {readlane_i32(os, at), readlane_i32(olen, at)};
  f->tile = readlane_i32(!causal ? k : QUERIES ? lo - 1 - (top - n) : n - lo, at);
  return true;
}

// A turn worked out beforehand (plan_kernel): tile < 0 is a turn without work.
struct alignas(32) Turn {
  Span own, other;
  int32_t tile;
  int32_t pad[3];
};

__device__ __forceinline__ bool find_planned(const Turn* turns, int32_t n, int32_t turn, Found* f) {
  const Turn* t = turns + rotated(turn, n);
  const i32x4 s = *reinterpret_cast<const i32x4*>(t);
  const int32_t tile = __builtin_amdgcn_readfirstlane(t->tile);
  f->own = {__builtin_amdgcn_readfirstlane(s[0]), __builtin_amdgcn_readfirstlane(s[1])};
  f->other = {__builtin_amdgcn_readfirstlane(s[2]), __builtin_amdgcn_readfirstlane(s[3])};
  f->tile = tile;
  return tile >= 0;
}

inline int64_t tile_turns(int64_t N, int64_t B, int bm) { return N / bm + B + 2; }

}  // namespace attn
}  // namespace mx
