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
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
struct Elem;

template <>
struct Elem<__bf16> {
  using x8 = bf16x8;
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

// A buffer descriptor of `bytes` bytes from a wave-uniform base: loads past
// them return zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}

__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}

// An offset no descriptor of ours covers.
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
// bytes, chunk c of row r at place c ^ f(r).  f spreads both kinds of reads
// over the banks: the row reads (lane l: chunk c of row l) and the transposing
// reads (16 lanes: 4 consecutive rows x 2 chunks).
template <int DP>
struct Tile {
  static constexpr int C = DP / 8;
  static constexpr int kRow = DP * 2;  // bytes

  static __device__ __forceinline__ int f(int r) {
    if constexpr (C == 16) return ((r & 7) << 1) | ((r >> 3) & 1);
    else if constexpr (C == 8) return ((r & 3) << 1) | ((r >> 2) & 1);
    else return (((r >> 1) & 1) << 1) | ((r >> 2) & 1);  // 4 and 12: rows 2i and 2i + 1 differ by 64 bytes
  }

  // Byte offset of chunk c of row r.
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ f(r)) << 4); }

  // Copies a tile of ROWS rows from global memory into LDS, without passing
  // through registers: THREADS threads, 16 bytes per lane and instruction, the
  // LDS side contiguous, the global side permuted.  Rows past the descriptor
  // and chunks past `d_chunks` become zeros.
  template <int ROWS, int THREADS>
  struct Loader {
    static constexpr int kAll = ROWS * C;  // 16-byte places
    static constexpr int kPer = kAll / THREADS;
    static_assert(kAll % THREADS == 0, "whole instructions");
    uint32_t off[kPer];

    __device__ __forceinline__ void init(int tid, uint32_t stride, int d_chunks) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int u = i * THREADS + tid;
        const int r = u / C, c = (u % C) ^ f(r);
        off[i] = c < d_chunks ? static_cast<uint32_t>(r) * stride + c * 16 : kOutside;
      }
    }

    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, char* lds, int wave) const {
#pragma unroll
      for (int i = 0; i < kPer; ++i) load16_to_lds(r, lds + (i * THREADS + wave * 64) * 16, off[i]);
    }
  };
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

// All LDS-direct loads of the wave have landed.
__device__ __forceinline__ void wait_lds_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// ---------------------------------------------------------------------------
// Packed lists
// ---------------------------------------------------------------------------
// Rows 0..N-1 are cut by B + 1 offsets.  Two more lists without partners hold
// the rows before the first and after the last offset (if there are any), so
// that every row belongs to one list: list 0 those before, lists 1..B the
// caller's, list B + 1 those after.  A launch needs the tiles of every list
// without a host copy of the offsets: list i owns the tile slots
// start(i) / BM + i up to start(i + 1) / BM + i + 1, which is at least
// ceil(length / BM) of them and N / BM + B + 2 in all, and a block finds its
// list by a search over those keys, 64 lists per step.

struct Span {
  int64_t start;
  int64_t len;  // >= 0
};

template <typename I>
__device__ __forceinline__ int64_t list_start(const I* offsets, int64_t B, int64_t N, int64_t i) {
  if (i <= 0) return 0;
  if (i > B + 1) return N;
  const int64_t o = static_cast<int64_t>(offsets[i - 1]);
  return o < 0 ? 0 : (o > N ? N : o);  // malformed offsets stay in bounds
}

template <typename I>
__device__ __forceinline__ Span list_span(const I* offsets, int64_t B, int64_t N, int64_t i) {
  const int64_t s = list_start(offsets, B, N, i), e = list_start(offsets, B, N, i + 1);
  return {s, e > s ? e - s : 0};
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(v >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// The list (0..B+1) that owns tile slot `slot`, and the tile's number in it.
template <typename I>
__device__ __forceinline__ int64_t find_list(const I* offsets, int64_t B, int64_t N, int bm_shift,
                                             int64_t slot, int64_t* tile) {
  int64_t lo = 0, n = B + 2;
  int64_t key = 0;
  while (n > 1) {
    const int64_t step = (n + 63) >> 6;
    const int64_t i = lo + lane_id() * step;
    const bool in = i < lo + n && (list_start(offsets, B, N, i) >> bm_shift) + i <= slot;
    const int c = __popcll(__ballot(in));  // the first lane's is always at most `slot`
    const int64_t at = (c > 0 ? c - 1 : 0) * step;
    lo += at;
    n = n - at < step ? n - at : step;
  }
  key = (list_start(offsets, B, N, lo) >> bm_shift) + lo;
  *tile = uniform64(slot - key);
  return uniform64(lo);
}

inline int64_t tile_slots(int64_t N, int64_t B, int bm) { return N / bm + B + 2; }

}  // namespace attn
}  // namespace mx
