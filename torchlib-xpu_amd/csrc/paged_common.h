// What the kernels of the paged key-value caches share: the cache and its pages,
// the list of a packed row, and how attention of one token per sequence is cut
// into shares and joined.
#pragma once

#include "attention_common.h"

namespace mx {
namespace attn {
namespace {

struct Cache {
  char *k, *v;
  int64_t k_page, k_slot, k_head;  // strides in bytes
  int64_t v_page, v_slot, v_head;
  const int32_t* table;
  int64_t table_row;               // stride of a sequence's row, in entries
  int64_t pages, width;            // pages of the cache; entries of a row
  int32_t page_size, page_shift;   // shift: log2 of a power of two, else -1
};

__device__ __forceinline__ int64_t ld_index(const void* p, int32_t bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i]
                    : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// Page of the table's row that holds token t (t >= 0), and its slot there.
__device__ __forceinline__ int64_t page_of(const Cache& c, int64_t t, int* slot) {
  const int64_t e = c.page_shift >= 0 ? t >> c.page_shift : t / c.page_size;
  *slot = static_cast<int>(t - e * c.page_size);
  return e;
}

// The last i of 0..B with offsets[i] <= row, or -1: 64 probes per step.
__device__ __forceinline__ int64_t list_of_row(const void* offsets, int32_t bytes, int64_t B, int64_t row) {
  int64_t lo = 0, n = B + 1;
  do {
    const int64_t step = (n + 63) >> 6;
    const int64_t i = lo + lane_id() * step;
    const bool in = i < lo + n && ld_index(offsets, bytes, i) <= row;
    const int c = __popcll(__ballot(in));
    if (c == 0) return -1;  // offsets[0] > row (a later step's first probe is known not to be)
    const int64_t at = (c - 1) * step;
    lo += at;
    n = n - at < step ? n - at : step;
  } while (n > 1);
  return uniform64(lo);
}

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane) {
  const uint32_t lo = __shfl(static_cast<int>(v), lane, 64);
  const uint32_t hi = __shfl(static_cast<int>(v >> 32), lane, 64);
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// ---------------------------------------------------------------------------
// Attention of one token per sequence
// ---------------------------------------------------------------------------

struct StepArgs {
  Cache c;
  const char* q;
  int64_t q_row, q_head;   // bytes
  const void* lengths;
  int32_t lengths_bytes;
  int32_t B, H, Hkv, G, D;
  int32_t head_blocks;     // of 16 query heads of a key-value head
  int32_t workers;         // per head block: they share all tiles; 0: a block per sequence
  int32_t wide;            // a block of 8 or 16 waves per sequence
  int32_t lead;            // of a share: what beginning a sequence costs, in tiles
  float scale;
  float units;             // of the running maximum, in base 2: scale log2(e), or 1
  void* out;               // [B, H, D]
  float* part;             // [workers, 2, H, D + 2]: sums, then maximum and sum of weights
};

constexpr int kStepWaves = 4;
constexpr int wide_waves(int D) { return D <= 64 ? 16 : 8; }  // by the registers
constexpr int kStepKeys = 32;  // keys of a wave's tile

// Tokens of sequence b that there are, and its tiles of 32 keys per wave of a block.
constexpr int kTileKeys = kStepWaves * kStepKeys;

__device__ __forceinline__ int32_t tokens_of(const StepArgs& a, int32_t b) {
  const int64_t n = ld_index(a.lengths, a.lengths_bytes, b), most = a.c.width * a.c.page_size;
  return static_cast<int32_t>(n < 0 ? 0 : (n < most ? n : most));
}
template <int WAVES = kStepWaves>
__device__ __forceinline__ int32_t tiles_of(int32_t tokens) {
  return (tokens + WAVES * kStepKeys - 1) / (WAVES * kStepKeys);
}

// The sequences' tiles end to end, each sequence's after `lead` units for its
// beginning, are cut into equal shares, one for a worker (and no more than units):
// share w begins at unit w total / shares.  A sequence's tiles may be cut anywhere;
// what a share has of one that it does not have whole is joined later.  Shares
// are equal whatever the lengths (a block per sequence waits for the longest).
__device__ __forceinline__ int64_t share_begin(int64_t w, int64_t total, int64_t shares) {
  return w * total / shares;
}
__device__ __forceinline__ int64_t share_of(int64_t unit, int64_t total, int64_t shares) {
  return ((unit + 1) * shares - 1) / total;
}
__device__ __forceinline__ int32_t units_of(const StepArgs& a, int32_t tokens) {
  return tokens > 0 ? tiles_of(tokens) + a.lead : 0;
}

// Units of all sequences, and of those before `b`.
__device__ __forceinline__ int64_t count_units(const StepArgs& a, int32_t b, int64_t* before) {
  int64_t all = 0, prior = 0;
  for (int32_t i0 = 0; i0 < a.B; i0 += 64) {
    const int32_t i = i0 + lane_id();
    const int32_t n = i < a.B ? units_of(a, tokens_of(a, i)) : 0;
    // 64 sequences of less than 2^24 units each.
    all += readlane_i32(wave_prefix(n), 63);
    if (i0 < b) prior += readlane_i32(wave_prefix(i < b ? n : 0), 63);
  }
  *before = prior;
  return all;
}

// A wave's place among the sequences: sequence b, and in lane i the tokens of
// sequence base + i (so that the next one costs no trip to memory).
struct Cursor {
  int32_t b, base, tokens;

  __device__ __forceinline__ void read(const StepArgs& a, int32_t from) {
    base = from;
    const int32_t i = base + lane_id();
    tokens = i < a.B ? tokens_of(a, i) : 0;
  }
  __device__ __forceinline__ int32_t length() const { return readlane_i32(tokens, b - base); }

  // On to the next sequence that has tokens; false if there is none.
  __device__ __forceinline__ bool next(const StepArgs& a) {
    int32_t from = b + 1;
    while (true) {
      const uint64_t left = from - base < 64 ? __ballot(tokens > 0) >> (from - base) << (from - base) : 0;
      if (left != 0) {
        b = base + __builtin_ctzll(left);
        return true;
      }
      from = base + 64;
      if (from >= a.B) return false;
      read(a, from);
    }
  }
};

// The share of `worker`: tiles [at, stop) counted from the first one of the cursor's
// sequence (`at` may lie before it).  False if there are fewer shares, or this one
// ends before a tile.
__device__ __forceinline__ bool find_share(const StepArgs& a, int worker, Cursor* c, int64_t* at, int64_t* stop) {
  int64_t prior;
  c->read(a, 0);
  const int64_t total = a.B <= 64 ? readlane_i32(wave_prefix(units_of(a, c->tokens)), 63) : count_units(a, 0, &prior);
  const int64_t shares = total < a.workers ? total : a.workers;  // none is empty
  if (worker >= shares) return false;
  int64_t from = share_begin(worker, total, shares), to = share_begin(worker + 1, total, shares);
  c->b = 0;
  for (int32_t i0 = 0; i0 < a.B; i0 += 64) {
    if (i0 > 0) c->read(a, i0);
    const int32_t upto = wave_prefix(units_of(a, c->tokens));
    const int32_t here = readlane_i32(upto, 63);
    if (from >= here) {
      from -= here;
      to -= here;
      continue;
    }
    const int l = __builtin_ctzll(__ballot(from < upto));
    c->b = i0 + l;
    const int32_t skip = readlane_i32(upto, l) - tiles_of(readlane_i32(c->tokens, l));  // its lead is behind it
    from -= skip;
    to -= skip;
    break;
  }
  *at = from;
  *stop = to;
  return to > 0;
}

// Joins what the block's waves have of sequence b's tiles [t0, t1) of n: the
// output, or this share's part of it.
template <typename T, int WAVES, int DP>
__device__ __forceinline__ void finish_block(const StepArgs& a, const float (&sh_o)[WAVES][16][DP + 1],
                                             const float (&sh_m)[WAVES][16], const float (&sh_l)[WAVES][16],
                                             int worker, int32_t b, int32_t t0, int32_t t1, int32_t n, int head0,
                                             int heads) {
  const float c2 = a.units;
  __syncthreads();
  const bool whole = t0 == 0 && t1 == n;
  for (int u = threadIdx.x; u < heads * a.D; u += WAVES * 64) {
    const int nh = u / a.D, d = u - nh * a.D;
    float mm = sh_m[0][nh];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, sh_m[w][nh]);
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = mm == -INFINITY ? 0.0f : exp2_hw((sh_m[w][nh] - mm) * c2);
      acc += f * sh_o[w][nh][d];
      l += f * sh_l[w][nh];
    }
    if (whole) {
      static_cast<T*>(a.out)[(static_cast<int64_t>(b) * a.H + head0 + nh) * a.D + d] =
          static_cast<T>(l == 0.0f ? 0.0f : acc / l);
    } else {
      // A sequence begun by an earlier share, or one that a later share ends.
      float* to = a.part + ((static_cast<int64_t>(worker) * 2 + (t0 > 0 ? 0 : 1)) * a.H + head0 + nh) * (a.D + 2);
      to[d] = acc;
      if (d == 0) {
        to[a.D] = mm;
        to[a.D + 1] = l;
      }
    }
  }
}

// Joins the shares of a sequence and head, in their order, and writes the
// sequences without tokens; one that a share had whole is written already.  With
// share s's maximum m_s, sum l_s and weighted values x_s, and m their largest
// maximum, the output is sum_s exp(m_s - m) x_s / sum_s exp(m_s - m) l_s.  A
// block per sequence and head: its waves take equal runs of the shares.  Bound:
// its launch and three loads in turn (5 us for 64 sequences of 32 heads).
constexpr int kJoinMost = 16;

template <typename T>
__global__ void __launch_bounds__(kJoinMost * 64) join_kernel(const StepArgs a) {
  __shared__ float sh_o[kJoinMost][MX_ATTENTION_MAX_D], sh_m[kJoinMost], sh_l[kJoinMost];
  const int32_t b = blockIdx.x / a.H, head = blockIdx.x % a.H;
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(blockIdx.x) * a.D;
  const int32_t n = __builtin_amdgcn_readfirstlane(tiles_of(tokens_of(a, b)));
  if (n == 0) {
    for (int d = threadIdx.x; d < a.D; d += blockDim.x) out[d] = static_cast<T>(0.0f);
    return;
  }
  int64_t before;
  const int64_t total = count_units(a, b, &before);
  const int64_t all = total < a.workers ? total : a.workers;
  before += a.lead;
  const int64_t w0 = share_of(before, total, all), w1 = share_of(before + n - 1, total, all);
  if (w0 == w1) return;
  const int shares = static_cast<int>(w1 - w0 + 1);
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = lane_id();
  const int from = shares * wave / waves, to = shares * (wave + 1) / waves;
  const float c2 = a.units;
  float m = -INFINITY, l = 0.0f, x0 = 0.0f, x1 = 0.0f;
  auto place = [&](int s) {
    return a.part + (((w0 + s) * 2 + (s == 0 ? 1 : 0)) * a.H + head) * (a.D + 2);
  };
  for (int s0 = from; s0 < to; s0 += 64) {
    const int k = to - s0 < 64 ? to - s0 : 64;
    float ms = -INFINITY, ls = 0.0f;
    if (lane < k) {
      const float* p = place(s0 + lane);
      ms = p[a.D];
      ls = p[a.D + 1];
    }
    float top = ms;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float m2 = fmaxf(m, top);
    const float base = m2 == -INFINITY ? 0.0f : m2;
    const float old = exp2_hw((m - base) * c2);
    const float f = exp2_hw((ms - base) * c2);
    l = l * old + wave_sum(f * ls);
    x0 *= old;
    x1 *= old;
    m = m2;
    for (int s = 0; s < k; s += 8) {  // 8 shares' sums asked for at once
      float v0[8], v1[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        v0[u] = v1[u] = 0.0f;
        if (s + u < k) {
          const float* p = place(s0 + s + u);
          if (lane < a.D) v0[u] = p[lane];
          if (lane + 64 < a.D) v1[u] = p[lane + 64];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float fs = __uint_as_float(readlane_i32(__float_as_uint(f), s + u));
        x0 += fs * v0[u];
        x1 += fs * v1[u];
      }
    }
  }
  sh_o[wave][lane] = x0;
  sh_o[wave][lane + 64] = x1;
  if (lane == 0) {
    sh_m[wave] = m;
    sh_l[wave] = l;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
    float mm = sh_m[0];
    for (int w = 1; w < waves; ++w) mm = fmaxf(mm, sh_m[w]);
    const float base = mm == -INFINITY ? 0.0f : mm;
    float acc = 0.0f, sum = 0.0f;
    for (int w = 0; w < waves; ++w) {
      const float f = exp2_hw((sh_m[w] - base) * c2);
      acc += f * sh_o[w][d];
      sum += f * sh_l[w];
    }
    out[d] = static_cast<T>(sum == 0.0f ? 0.0f : acc / sum);
  }
}

inline int32_t head_blocks_of(int32_t H, int32_t Hkv) { return static_cast<int32_t>(ceil_div(H / Hkv, 16)); }

// What caches of 16-bit values and of 4-bit rows (bytes) have to fulfil.
inline int check_rows_cache(const mx_paged_cache* c, int32_t bits) {
  MX_REQUIRE(c != nullptr, "cache is null");
  MX_REQUIRE(bits == 16 || bits == 4, "%d bits: a cache has 16 or 4", bits);
  MX_REQUIRE(c->page_size > 0 && c->pages >= 0 && c->table_width >= 0, "bad page or table size");
  MX_REQUIRE(c->pages == 0 || (c->k != nullptr && c->v != nullptr), "cache tensors are null");
  const int align = bits == 16 ? 16 : 4, step = bits == 16 ? 8 : 4;
  for (const void* p : {static_cast<const void*>(c->k), static_cast<const void*>(c->v)})
    MX_REQUIRE(reinterpret_cast<uintptr_t>(p) % align == 0, "cache tensors must be %d-byte aligned", align);
  for (int64_t s : {c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->v_page_stride, c->v_slot_stride,
                    c->v_head_stride})
    MX_REQUIRE(s >= 0 && s % step == 0, "cache strides must be multiples of %d elements", step);
  return MX_OK;
}

// `bytes`: of an element of the cache, in which its strides are counted.
inline Cache cache_of(const mx_paged_cache* c, int64_t bytes) {
  Cache x{};
  x.k = static_cast<char*>(c->k);
  x.v = static_cast<char*>(c->v);
  x.k_page = c->k_page_stride * bytes, x.k_slot = c->k_slot_stride * bytes, x.k_head = c->k_head_stride * bytes;
  x.v_page = c->v_page_stride * bytes, x.v_slot = c->v_slot_stride * bytes, x.v_head = c->v_head_stride * bytes;
  x.table = c->table;
  x.table_row = c->table_row_stride;
  x.pages = c->pages;
  x.width = c->pages > 0 ? c->table_width : 0;  // no page, no token
  x.page_size = c->page_size;
  x.page_shift = -1;
  if ((c->page_size & (c->page_size - 1)) == 0) x.page_shift = __builtin_ctz(c->page_size);
  return x;
}

}  // namespace
}  // namespace attn
}  // namespace mx
