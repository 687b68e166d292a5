// A paged key-value cache: writing packed rows into it, and attention of one
// new token per sequence over it.
//
// Token t of sequence b lives in slot t % page_size of page
// table[b, t / page_size].  A page number outside [0, pages) is never
// followed: an append drops the row, the attention takes the token as absent.
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

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------

struct AppendArgs {
  Cache c;
  const char *k, *v;
  int64_t k_row, k_head, v_row, v_head;  // bytes
  const void *offsets, *starts;
  int32_t offsets_bytes, starts_bytes;
  int64_t B, N;
  int32_t Hkv, chunks;                   // 16-byte chunks of a head
};

// The last i of 0..B with offsets[i] <= row, or -1: 64 probes per step.
__device__ __forceinline__ int64_t list_of_row(const void* offsets, int32_t bytes, int64_t B, int64_t row) {
  int64_t lo = 0, n = B + 1;
  if (ld_index(offsets, bytes, 0) > row) return -1;
  while (n > 1) {
    const int64_t step = (n + 63) >> 6;
    const int64_t i = lo + lane_id() * step;
    const bool in = i < lo + n && ld_index(offsets, bytes, i) <= row;
    const int c = __popcll(__ballot(in));
    const int64_t at = (c > 0 ? c - 1 : 0) * step;
    lo += at;
    n = n - at < step ? n - at : step;
  }
  return uniform64(lo);
}

constexpr int kAppendWaves = 4;

// A wave per row: it finds the row's list and page, then copies the row's
// heads of both tensors in 16-byte chunks.  Bound: the copy (32 lists of 1 to
// 2000 rows, 8 heads of 128: 52 us, 5.0 TB/s read and written); few rows by the
// three loads in turn before it (64 rows: 4.9 us, of which the launch 3.5).
__global__ void __launch_bounds__(kAppendWaves * 64) append_kernel(const AppendArgs a) {
  const int64_t row = uniform64(static_cast<int64_t>(blockIdx.x) * kAppendWaves + (threadIdx.x >> 6));
  if (row >= a.N) return;
  const int64_t b = list_of_row(a.offsets, a.offsets_bytes, a.B, row);
  if (b < 0 || b >= a.B) return;
  const int64_t start = ld_index(a.starts, a.starts_bytes, b);
  const int64_t t = start + row - ld_index(a.offsets, a.offsets_bytes, b);
  if (start < 0 || t < 0) return;
  int slot;
  const int64_t e = page_of(a.c, t, &slot);
  if (e >= a.c.width) return;
  const int64_t page = a.c.table[b * a.c.table_row + e];
  if (page < 0 || page >= a.c.pages) return;
  const char* ks = a.k + row * a.k_row;
  const char* vs = a.v + row * a.v_row;
  char* kd = a.c.k + page * a.c.k_page + slot * a.c.k_slot;
  char* vd = a.c.v + page * a.c.v_page + slot * a.c.v_slot;
  const int n = a.Hkv * a.chunks;
  for (int u = lane_id(); u < n; u += 64) {
    const int h = u / a.chunks, c = u - h * a.chunks;
    const i32x4 x = *reinterpret_cast<const i32x4*>(ks + h * a.k_head + c * 16);
    const i32x4 y = *reinterpret_cast<const i32x4*>(vs + h * a.v_head + c * 16);
    *reinterpret_cast<i32x4*>(kd + h * a.c.k_head + c * 16) = x;
    *reinterpret_cast<i32x4*>(vd + h * a.c.v_head + c * 16) = y;
  }
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
  float scale;
  void* out;               // [B, H, D]
  float* part;             // [workers, 2, H, D + 2]: sums, then maximum and sum of weights
};

constexpr int kStepWaves = 4;
constexpr int wide_waves(int D) { return D <= 64 ? 16 : 8; }  // by the registers
constexpr int kStepKeys = 32;  // keys of a wave's tile

// N values of 16 bits from global memory.
template <int N>
struct Piece;
template <>
struct Piece<2> { using type = int; };
template <>
struct Piece<4> { using type = i32x2; };
template <>
struct Piece<8> { using type = i32x4; };

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane) {
  const uint32_t lo = __shfl(static_cast<int>(v), lane, 64);
  const uint32_t hi = __shfl(static_cast<int>(v >> 32), lane, 64);
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

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

// The sequences' tiles end to end are cut into equal shares, one for a worker
// (and no more than tiles): share w begins at tile w total / shares.  A sequence's tiles may be cut anywhere;
// what a share has of one that it does not have whole is joined later.  Shares
// are equal whatever the lengths (a block per sequence waits for the longest).
__device__ __forceinline__ int64_t share_begin(int64_t w, int64_t total, int64_t shares) {
  return w * total / shares;
}
__device__ __forceinline__ int64_t share_of(int64_t tile, int64_t total, int64_t shares) {
  return ((tile + 1) * shares - 1) / total;
}

// Tiles of all sequences, and of those before `b`.
__device__ __forceinline__ int64_t count_tiles(const StepArgs& a, int32_t b, int64_t* before) {
  int64_t all = 0, prior = 0;
  for (int32_t i0 = 0; i0 < a.B; i0 += 64) {
    const int32_t i = i0 + lane_id();
    const int32_t n = i < a.B ? tiles_of(tokens_of(a, i)) : 0;
    // 64 sequences of less than 2^24 tiles each.
    all += readlane_i32(wave_prefix(n), 63);
    if (i0 < b) prior += readlane_i32(wave_prefix(i < b ? n : 0), 63);
  }
  *before = prior;
  return all;
}

// One block: up to 16 query heads of one key-value head, and a share of its
// tiles (or one sequence); its waves take 32 of a tile's keys each.  Every
// key and value is read once, straight into registers in the matrix operands'
// layouts (r = lane % 16, g = lane / 16): 16 keys x 32 columns of K per 16x16x32
// product, a head per result column; 8 keys and DP / 16 columns of V per lane,
// transposed in registers (a value is used once: through LDS it would cost a
// write and a read more, and hold up its wave).  A maximum m and a sum of
// exp(s - m) per head run along, as for whole prompts; the waves' are joined
// through LDS.  Probabilities are rounded to the cache's type for the second
// product; scores, sums and the running maximum are fp32.
//
// Bound: reading the cache (256 sequences of 8192, 16 heads of 128 over 4: 743 us,
// 5.8 TB/s; 64 of 1 to 4096, 32 heads over 8: 106 us, 5.1 TB/s, of which 5 us the
// join); one short sequence by latency (777 tokens, 8 heads of 64: 8.4 us: the
// launch, length, table and two tiles of keys in turn).
template <typename T, int DP, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, WAVES == kStepWaves ? 2 : WAVES / 4) step_kernel(const StepArgs a) {
  using E = Elem<T>;
  using X8 = typename E::x8;
  constexpr int kTile = WAVES * kStepKeys;
  constexpr int KS = DP / 32;  // products along D of a score
  constexpr int EV = DP / 16;  // columns of V per lane
  using VP = typename Piece<EV>::type;
  __shared__ float sh_o[WAVES][16][DP + 1];
  __shared__ float sh_m[WAVES][16], sh_l[WAVES][16];

  const int heads_all = a.Hkv * a.head_blocks;
  const int hh = blockIdx.x % heads_all, worker = blockIdx.x / heads_all;
  const int kvh = hh / a.head_blocks, hb = hh % a.head_blocks;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int head0 = kvh * a.G + hb * 16;
  const int heads = a.G - hb * 16 < 16 ? a.G - hb * 16 : 16;
  const float c2 = a.scale * kLog2e;
  const char* kb = a.c.k + kvh * a.c.k_head;
  const char* vb = a.c.v + kvh * a.c.v_head;

  // The share: tiles [at, stop) counted from sequence b's first one.
  const bool shared = WAVES == kStepWaves && a.workers > 0;
  int32_t b = worker, len;
  int64_t at = 0, stop = 0;
  if (!shared) {
    len = __builtin_amdgcn_readfirstlane(tokens_of(a, b));
    stop = tiles_of<WAVES>(len);  // 0 for an empty one: its one pass writes the zeros
  } else {
    int64_t prior;
    const int64_t total = count_tiles(a, 0, &prior);
    const int64_t shares = total < a.workers ? total : a.workers;  // none is empty
    if (worker >= shares) return;
    at = share_begin(worker, total, shares);
    stop = share_begin(worker + 1, total, shares);
    len = 0;
    for (int32_t i0 = 0; i0 < a.B; i0 += 64) {
      const int32_t i = i0 + lane_id();
      const int32_t tokens = i < a.B ? tokens_of(a, i) : 0;
      const int32_t upto = wave_prefix(tiles_of<WAVES>(tokens));
      const int32_t here = readlane_i32(upto, 63);
      if (at >= here) {
        at -= here;
        stop -= here;
        continue;
      }
      const int l = __builtin_ctzll(__ballot(at < upto));
      b = i0 + l;
      len = readlane_i32(tokens, l);
      const int32_t skip = readlane_i32(upto, l) - tiles_of<WAVES>(len);
      at -= skip;
      stop -= skip;
      break;
    }
  }

  while (true) {
    const int32_t n = tiles_of<WAVES>(len);
    const int32_t t0 = static_cast<int32_t>(at), t1 = static_cast<int32_t>(stop < n ? stop : n);
    const int32_t end = t1 * kTile < len ? t1 * kTile : len;

    X8 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int col = 32 * s + 8 * g;
      i32x4 w{};
      if (r < heads && col < a.D)
        w = *reinterpret_cast<const i32x4*>(a.q + b * a.q_row + (head0 + r) * a.q_head + col * 2);
      qf[s] = __builtin_bit_cast(X8, w);
    }
    float m = -INFINITY, sum = 0.0f;
    f32x4 o[EV];
#pragma unroll
    for (int t = 0; t < EV; ++t) o[t] = f32x4{};

    // Lane i finds the place of key i % 32 of a tile; the table's entries of
    // the next tile are asked for before this one's keys.
    const int32_t* row = a.c.table + b * a.c.table_row;
    auto entry = [&](int32_t k0, int* slot) {
      const uint32_t key = k0 + (lane & 31);
      const uint32_t size = a.c.page_size;
      const uint32_t e = a.c.page_shift >= 0 ? key >> a.c.page_shift : key / size;
      *slot = static_cast<int>(key - e * size);
      return key < static_cast<uint32_t>(end) ? row[e] : -1;
    };
    const int32_t first = t0 * kTile + wave * kStepKeys;
    int slot_next = 0;
    int32_t page_next = entry(first, &slot_next);
    for (int32_t k0 = first; k0 < end; k0 += kTile) {
      const int64_t page = page_next;
      const int slot = slot_next;
      page_next = entry(k0 + kTile, &slot_next);
      const bool there = page >= 0 && page < a.c.pages;
      const uint32_t seen = static_cast<uint32_t>(__ballot(there));
      const int64_t koff = there ? page * a.c.k_page + slot * a.c.k_slot : 0;
      const int64_t voff = there ? page * a.c.v_page + slot * a.c.v_slot : 0;

      i32x4 kw[2][KS];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const char* p = kb + shfl64(koff, 16 * u + r);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int col = 32 * s + 8 * g;
          kw[u][s] = i32x4{};
          if (col < a.D) kw[u][s] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p + col * 2));
        }
      }
      VP vw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int nk = 16 * (i / 4) + 4 * g + i % 4;
        const char* p = vb + shfl64(voff, nk);
        vw[i] = VP{};
        if (EV * r < a.D && ((seen >> nk) & 1)) vw[i] = __builtin_nontemporal_load(reinterpret_cast<const VP*>(p + EV * r * 2));
      }

      f32x4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = f32x4{};
#pragma unroll
        for (int x = 0; x < KS; ++x) s[u] = E::mfma16(__builtin_bit_cast(X8, kw[u][x]), qf[x], s[u]);
      }
      if (seen != 0xffffffffu) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (((seen >> (16 * u + 4 * g + i)) & 1) == 0) s[u][i] = -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                        fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      if (__any((top - m) * c2 > 8.0f)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, other_half(top));
        const float m2 = fmaxf(m, top);
        const float f = m2 == -INFINITY ? 1.0f : exp2_hw((m - m2) * c2);
        sum *= f;
#pragma unroll
        for (int t = 0; t < EV; ++t) o[t] *= f;
        m = m2;
      }
      const float mc = m == -INFINITY ? 0.0f : m * c2;
      X8 p;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = exp2_hw(__builtin_fmaf(s[i / 4][i % 4], c2, -mc));
        sum += e;
        p[i] = static_cast<T>(e);
      }
      typedef T TV __attribute__((ext_vector_type(EV)));
#pragma unroll
      for (int t = 0; t < EV; ++t) {
        X8 vt;
#pragma unroll
        for (int i = 0; i < 8; ++i) vt[i] = __builtin_bit_cast(TV, vw[i])[t];
        o[t] = E::mfma16(vt, p, o[t]);
      }
    }

    // The waves' sums: lane (r, g) holds head r, columns EV (4 g + i) + t.
    sum += __shfl_xor(sum, 16, 64);
    sum += other_half(sum);
    if (g == 0) {
      sh_m[wave][r] = m;
      sh_l[wave][r] = sum;
    }
#pragma unroll
    for (int t = 0; t < EV; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sh_o[wave][r][EV * (4 * g + i) + t] = o[t][i];
    __syncthreads();
    const bool whole = t0 == 0 && t1 == n;
    for (int u = tid; u < heads * a.D; u += WAVES * 64) {
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
    if (!shared || stop <= n) return;  // a block per sequence never leaves its own
    // The next sequence that has tokens.
    stop -= n;
    at = 0;
    do {
      ++b;
      len = __builtin_amdgcn_readfirstlane(tokens_of(a, b));
    } while (len == 0 && b + 1 < a.B);
    if (len == 0) return;
    __syncthreads();
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
  const int64_t total = count_tiles(a, b, &before);
  const int64_t all = total < a.workers ? total : a.workers;
  const int64_t w0 = share_of(before, total, all), w1 = share_of(before + n - 1, total, all);
  if (w0 == w1) return;
  const int shares = static_cast<int>(w1 - w0 + 1);
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = lane_id();
  const int from = shares * wave / waves, to = shares * (wave + 1) / waves;
  const float c2 = a.scale * kLog2e;
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

// How a call's sequences are cut.  Times in us, of back-to-back calls with an
// event on both sides (about 5 of them the launch).
// - Workers that share all tiles, two blocks for every CU (64 ragged sequences of
//   up to 4096 tokens, 8 x 128: a block per sequence in halves 147, shares with
//   one, two and three blocks a CU 119, 106 and 122).  What they leave is joined
//   by a second launch, which waits for the first.
// - Where no sequence can have more than two tiles of a wide block (8 or 16
//   waves), and blocks are few enough to start nearly at once, such a block per
//   sequence and head instead of the second launch (8 heads of 64: one sequence
//   of 777 15.2 -> 11.1, of 2048 15.5 -> 17.8; 64 of up to 1024 31.1 -> 27.4; 200
//   of up to 1024 70.3 -> 70.9; 8 heads of 128: 64 of up to 512 29.6 -> 25.4, 200
//   57.7 -> 63.4).
// - A block of four waves per sequence and head where these are enough to even
//   out by themselves, or no sequence has two tiles.  The host knows no lengths, and
//   lengths decide: this way gains where they are alike or short (1024 of up to 200
//   tokens, 8 x 64: 72, in shares 110; 256 of 8192, 8 x 64: 903, in shares 1000; 512
//   of 1 to 1000 by their logarithm, 4 x 64: 38, in shares 41) and loses where few are
//   long (256 of up to 2000, 8 x 128: 211, in shares 201; by their logarithm 90, in
//   shares 70; up to 8192 by their logarithm 298, in shares 184).
struct Plan {
  int32_t workers;  // 0: a block per sequence and head
  bool wide;
};

Plan plan_step(int64_t B, int32_t heads, int32_t D, int64_t most) {
  const int64_t tiles = ceil_div(most, kTileKeys), blocks = B * heads, cus = num_cus();
  if (tiles <= 1 || blocks >= 8 * cus) return {0, false};
  if (most <= 2 * wide_waves(D) * kStepKeys && blocks <= 4 * cus) return {0, true};
  const int64_t w = ceil_div(cus * 2, heads);
  return {static_cast<int32_t>(w < B * tiles ? w : B * tiles), false};
}

int32_t head_blocks_of(int32_t H, int32_t Hkv) { return static_cast<int32_t>(ceil_div(H / Hkv, 16)); }

int check_cache(const mx_paged_cache* c, int32_t dtype, int32_t Hkv, int32_t D) {
  MX_REQUIRE(c != nullptr, "cache is null");
  MX_REQUIRE(dtype == MX_DTYPE_F16 || dtype == MX_DTYPE_BF16, "dtype %d is not fp16 or bf16", dtype);
  MX_REQUIRE(Hkv > 0 && D > 0 && D % 8 == 0 && D <= MX_ATTENTION_MAX_D,
             "head width %d is no multiple of 8 up to %d", D, MX_ATTENTION_MAX_D);
  MX_REQUIRE(c->page_size > 0 && c->pages >= 0 && c->table_width >= 0, "bad page or table size");
  MX_REQUIRE(c->pages == 0 || (c->k != nullptr && c->v != nullptr), "cache tensors are null");
  for (const void* p : {static_cast<const void*>(c->k), static_cast<const void*>(c->v)})
    MX_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "cache tensors must be 16-byte aligned");
  for (int64_t s : {c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->v_page_stride,
                    c->v_slot_stride, c->v_head_stride})
    MX_REQUIRE(s >= 0 && s % 8 == 0, "cache strides must be multiples of 8 elements");
  return MX_OK;
}

Cache cache_of(const mx_paged_cache* c) {
  Cache x{};
  x.k = static_cast<char*>(c->k);
  x.v = static_cast<char*>(c->v);
  x.k_page = c->k_page_stride * 2, x.k_slot = c->k_slot_stride * 2, x.k_head = c->k_head_stride * 2;
  x.v_page = c->v_page_stride * 2, x.v_slot = c->v_slot_stride * 2, x.v_head = c->v_head_stride * 2;
  x.table = c->table;
  x.table_row = c->table_row_stride;
  x.pages = c->pages;
  x.width = c->pages > 0 ? c->table_width : 0;  // no page, no token
  x.page_size = c->page_size;
  x.page_shift = -1;
  if ((c->page_size & (c->page_size - 1)) == 0) x.page_shift = __builtin_ctz(c->page_size);
  return x;
}

template <typename T, int DP>
int launch_step(const StepArgs& a, hipStream_t s) {
  const int64_t blocks = static_cast<int64_t>(a.workers > 0 ? a.workers : a.B) * a.Hkv * a.head_blocks;
  const int64_t joins = static_cast<int64_t>(a.B) * a.H;
  MX_REQUIRE(blocks < (1ll << 22) && joins < (1ll << 22), "too many sequences: %d", a.B);  // threads in 32 bits
  if (a.wide)
    step_kernel<T, DP, wide_waves(DP)><<<dim3(static_cast<unsigned>(blocks)), wide_waves(DP) * 64, 0, s>>>(a);
  else
    step_kernel<T, DP, kStepWaves><<<dim3(static_cast<unsigned>(blocks)), kStepWaves * 64, 0, s>>>(a);
  if (a.workers > 0) {
    const int waves = a.workers / a.B < 8 ? 1 : a.workers / a.B < 32 ? 4 : kJoinMost;
    join_kernel<T><<<dim3(static_cast<unsigned>(joins)), waves * 64, 0, s>>>(a);
  }
  MX_LAUNCH_CHECK();
  return MX_OK;
}

template <typename T>
int step_by_width(const StepArgs& a, hipStream_t s) {
  if (a.D <= 32) return launch_step<T, 32>(a, s);
  if (a.D <= 64) return launch_step<T, 64>(a, s);
  return launch_step<T, 128>(a, s);
}

}  // namespace
}  // namespace attn
}  // namespace mx

extern "C" int mx_paged_cache_append(const mx_paged_cache* cache, int32_t dtype, int32_t Hkv, int32_t D,
                                     const mx_attention_tensor* k, const mx_attention_tensor* v,
                                     int64_t N, int64_t B, const void* offsets,
                                     int32_t offsets_bytes, const void* starts,
                                     int32_t starts_bytes, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_cache(cache, dtype, Hkv, D)) return rc;
  MX_REQUIRE(N >= 0 && B >= 0, "negative size");
  if (N == 0 || B == 0 || cache->pages == 0 || cache->table_width == 0) return MX_OK;
  MX_REQUIRE(k != nullptr && v != nullptr && k->data != nullptr && v->data != nullptr &&
                 offsets != nullptr && starts != nullptr && cache->table != nullptr,
             "null argument");
  MX_REQUIRE((offsets_bytes == 4 || offsets_bytes == 8) && (starts_bytes == 4 || starts_bytes == 8),
             "index bytes %d and %d", offsets_bytes, starts_bytes);
  for (const mx_attention_tensor* t : {k, v})
    MX_REQUIRE(reinterpret_cast<uintptr_t>(t->data) % 16 == 0 && t->row_stride % 8 == 0 &&
                   t->head_stride % 8 == 0 && t->row_stride >= 0 && t->head_stride >= 0,
               "k and v: rows and heads must start at multiples of 16 bytes");
  AppendArgs a{};
  a.c = cache_of(cache);
  a.k = static_cast<const char*>(k->data);
  a.v = static_cast<const char*>(v->data);
  a.k_row = k->row_stride * 2, a.k_head = k->head_stride * 2;
  a.v_row = v->row_stride * 2, a.v_head = v->head_stride * 2;
  a.offsets = offsets, a.starts = starts;
  a.offsets_bytes = offsets_bytes, a.starts_bytes = starts_bytes;
  a.B = B, a.N = N;
  a.Hkv = Hkv, a.chunks = D / 8;
  const int64_t blocks = mx::ceil_div(N, kAppendWaves);
  MX_REQUIRE(blocks < (1ll << 24), "too many rows: %lld", (long long)N);  // threads in 32 bits
  append_kernel<<<dim3(static_cast<unsigned>(blocks)), kAppendWaves * 64, 0, mx::as_stream(stream)>>>(a);
  MX_LAUNCH_CHECK();
  return MX_OK;
}

extern "C" size_t mx_paged_cache_attention_workspace_bytes(const mx_paged_cache* cache, int64_t B,
                                                           int32_t H, int32_t Hkv, int32_t D) {
  using namespace mx::attn;
  if (cache == nullptr || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0) return 0;
  const Plan plan = plan_step(B, Hkv * head_blocks_of(H, Hkv), D, cache->table_width * cache->page_size);
  return static_cast<size_t>(plan.workers) * 2 * H * (D + 2) * sizeof(float);
}

extern "C" int mx_paged_cache_attention(const mx_paged_cache* cache, int32_t dtype,
                                        const mx_attention_tensor* q, int64_t B, int32_t H,
                                        int32_t Hkv, int32_t D, const void* lengths,
                                        int32_t lengths_bytes, float scale, void* out,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_cache(cache, dtype, Hkv, D)) return rc;
  MX_REQUIRE(B >= 0 && B < (1ll << 31), "%lld sequences", (long long)B);
  MX_REQUIRE(cache->table_width <= (1ll << 30) / cache->page_size, "more than 2^30 tokens in a row of the table");
  MX_REQUIRE(H > 0 && H % Hkv == 0, "%d query heads are no multiple of %d key-value heads", H, Hkv);
  MX_REQUIRE(std::isfinite(scale) && scale > 0.0f, "scale must be positive and finite");
  MX_REQUIRE(lengths_bytes == 4 || lengths_bytes == 8, "lengths_bytes %d", lengths_bytes);
  if (B == 0) return MX_OK;
  MX_REQUIRE(q != nullptr && q->data != nullptr && out != nullptr && lengths != nullptr &&
                 (cache->table != nullptr || cache->table_width == 0),
             "null argument");
  MX_REQUIRE(reinterpret_cast<uintptr_t>(q->data) % 16 == 0 && q->row_stride % 8 == 0 &&
                 q->head_stride % 8 == 0 && q->row_stride >= 0 && q->head_stride >= 0,
             "q: rows and heads must start at multiples of 16 bytes");
  StepArgs a{};
  a.c = cache_of(cache);
  a.q = static_cast<const char*>(q->data);
  a.q_row = q->row_stride * 2, a.q_head = q->head_stride * 2;
  a.lengths = lengths, a.lengths_bytes = lengths_bytes;
  a.B = static_cast<int32_t>(B), a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.D = D;
  a.head_blocks = head_blocks_of(H, Hkv);
  a.scale = scale;
  a.out = out;
  const Plan plan = plan_step(B, Hkv * a.head_blocks, D, cache->table_width * cache->page_size);
  a.workers = plan.workers, a.wide = plan.wide;
  const size_t need = mx_paged_cache_attention_workspace_bytes(cache, B, H, Hkv, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return mx::set_error(MX_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = mx::as_stream(stream);
  return dtype == MX_DTYPE_BF16 ? step_by_width<__bf16>(a, s) : step_by_width<_Float16>(a, s);
}
