// Attention over packed (jagged) sequences, forward and backward, for fp16 and
// bf16 with grouped key-value heads.
//
// List b has queries i in [0, Lq) and keys j in [0, Lk); query i sees key j if
// !causal or j <= i + Lk - Lq (the last query sees every key).  Over the
// visible keys
//   s_ij = scale q_i.k_j,  lse_i = log sum_j exp(s_ij),  p_ij = exp(s_ij - lse_i),
//   o_i = sum_j p_ij v_j;   a query that sees no key has o_i = 0, lse_i = -inf.
#include "attention_common.h"
#include <algorithm>

namespace mx {
namespace attn {
namespace {

constexpr int kBN = 64;        // keys per tile
constexpr int kRowWaves = 4;   // waves of 32 queries: tiles of 128, of one head
constexpr int kRowShift = 7;

struct PlanArgs {
  const void *q_offsets, *k_offsets;
  int32_t B, Nq, Nk, causal;
  Turn* turns[2];                  // of the queries' tiles and the keys' tiles
  int32_t n[2];
  int32_t shift[2];                // log2 of a tile's rows
};

// The order of a launch's tiles where lists are many and long: list by list, those
// with the most partners first (a block's time is its tile's length: the longest
// must not start last), a list's tiles one after another, as they read the same
// keys.  Block 0 orders the queries' tiles, block 1 the keys'.  The lists are
// counted into bins by the leading bits of their partners' number (exponent and 5
// more: 3%), whose sums are the bins' first turns; order within a bin is as it
// comes, which decides when a tile is worked on, never what comes out.
constexpr int kPlanThreads = 1024;  // and as many bins

template <typename I>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  __shared__ int32_t bins[kPlanThreads], sums[kPlanThreads / 64];
  const bool keys = blockIdx.x == 1;
  const I* own = static_cast<const I*>(keys ? a.k_offsets : a.q_offsets);
  const I* other = static_cast<const I*>(keys ? a.q_offsets : a.k_offsets);
  const int32_t N = keys ? a.Nk : a.Nq, Nother = keys ? a.Nq : a.Nk;
  Turn* turns = a.turns[blockIdx.x];
  const int32_t most = a.n[blockIdx.x], shift = a.shift[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  struct List { Span own, other; int32_t tiles, bin; };
  auto list = [&](int32_t i) {
    List x{};
    if (i > a.B + 1) return x;
    const int32_t s = list_start(own, a.B, N, i), e = list_start(own, a.B, N, i + 1);
    const int32_t os = list_start(other, a.B, Nother, i), oe = list_start(other, a.B, Nother, i + 1);
    x.own = {s, e > s ? e - s : 0};
    x.other = {os, i > 0 && i <= a.B && oe > os ? oe - os : 0};
    x.tiles = (x.own.len + (1 << shift) - 1) >> shift;
    // 2^0 .. 2^22 partners: bins 736 .. 1 from the end.
    const int32_t bits = static_cast<int32_t>(__float_as_uint(static_cast<float>(x.other.len)) >> 18) - (127 << 5) + 1;
    x.bin = kPlanThreads - 1 - (bits > 0 ? bits : 0);
    return x;
  };

  bins[tid] = 0;
  const List first = list(tid);
  __syncthreads();
  for (int32_t i = tid; i <= a.B + 1; i += kPlanThreads) {
    const List x = i == tid ? first : list(i);
    if (x.tiles > 0) atomicAdd(&bins[x.bin], x.tiles);
  }
  __syncthreads();
  const int32_t here = bins[tid];
  int32_t before = wave_prefix(here);
  if (lane == 63) sums[wave] = before;
  __syncthreads();
  int32_t total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w == wave) before += total;
    total += sums[w];
  }
  bins[tid] = before - here;
  __syncthreads();
  for (int32_t i = tid; i <= a.B + 1; i += kPlanThreads) {
    const List x = i == tid ? first : list(i);
    if (x.tiles == 0) continue;
    const int32_t at = atomicAdd(&bins[x.bin], x.tiles);
    for (int32_t t = 0; t < x.tiles; ++t) {
      if (static_cast<uint32_t>(at + t) >= static_cast<uint32_t>(most)) break;  // offsets that decrease: more tiles than turns
      Turn w{};
      w.own = x.own;
      w.other = x.other;
      w.tile = keys || !a.causal ? t : x.tiles - 1 - t;
      turns[at + t] = w;
    }
  }
  for (int64_t t = int64_t{total < 0 ? 0 : total} + tid; t < most; t += kPlanThreads) turns[t].tile = -1;
}

struct FwdArgs {
  const char *q, *k, *v;           // bytes
  uint32_t q_row, k_row, v_row;    // strides in bytes (at most 2^24)
  int64_t q_head, k_head, v_head;
  const void *q_offsets, *k_offsets;
  int32_t B, Nq, Nk;
  int32_t H, G, D;                 // G query heads per key-value head
  int32_t causal;
  int32_t pack;                    // log2 of the heads of a block
  int32_t ranked;                  // find_ranked finds the tiles
  const Turn* turns;               // find_planned does, among n_turns, if not null
  int32_t n_turns;
  float scale;
  void* out;                       // [Nq, H, D]
  float* lse;                      // [H, Nq] or null
};

// Which head a block works on, and which of its tiles (the 0th first).  Blocks
// go to the 8 XCDs in turn: with a multiple of 8 heads each XCD keeps H / 8
// neighbouring heads (which share keys) and takes all their tiles, so its L2
// holds few keys and the causal tiles, unequal in length, spread evenly.
__device__ __forceinline__ void head_and_turn(uint32_t bid, uint32_t H, int* head, int* turn) {
  if (H % 8 == 0) {
    const uint32_t per = H / 8, x = bid % 8, y = bid / 8;
    *head = x * per + y % per;
    *turn = y / per;
  } else {
    *head = bid % H;
    *turn = bid / H;
  }
}

// Writes a transposed result: column l of acc, scaled and rounded to the
// output's type, is row l (of `rows`) at `base` of a contiguous [.., heads, D].
template <typename T, int DP>
__device__ __forceinline__ void store_rows(void* base, const f32x16* acc, float scale, int rows,
                                           int heads, int D, int l, int h) {
  typedef T x4 __attribute__((ext_vector_type(4)));
  const uint32_t stride = static_cast<uint32_t>(heads) * D * 2;
  const __amdgpu_buffer_rsrc_t r = make_rsrc(base, span_bytes(rows, stride, D * 2));
  const uint32_t row = l < rows ? l * stride + h * 8 : kOutside;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i / 4);  // and 4 more from the other half-wave: D is a multiple of 8
      x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(acc[d][i + e] * scale);
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, w), r, col < D ? row + col * 2 : kOutside, 0, 0);
    }
}

// The same unscaled in fp32, at `base` of a contiguous [.., heads, D].
template <int DP>
__device__ __forceinline__ void store_sums(float* base, const f32x16* acc, int rows, int heads, int D,
                                           int l, int h) {
  if (l >= rows) return;
  float* row = base + int64_t{l} * heads * D + 4 * h;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i / 4);
      if (col < D) *reinterpret_cast<f32x4*>(row + col) = f32x4{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
    }
}

// Row l of a 32-row tile as the B operand: 8 columns per step.
template <typename X8, int KS>
__device__ __forceinline__ void load_rows(X8* f, const char* base, int rows, int64_t stride, int D,
                                          int l, int h) {
  const __amdgpu_buffer_rsrc_t r = make_rsrc(base, span_bytes(rows, static_cast<uint32_t>(stride), D * 2));
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int c = 2 * s + h;
    const uint32_t off = c * 8 < D ? static_cast<uint32_t>(l) * static_cast<uint32_t>(stride) + c * 16 : kOutside;
    f[s] = __builtin_bit_cast(X8, load16(r, off));
  }
}


// This lane's row f (its half of the columns) times the row at p, summed over
// both half-waves.
template <int DP, typename X8>
__device__ __forceinline__ float dot_row(const X8* f, const char* p, int D, int h) {
  float s = 0.0f;
#pragma unroll
  for (int x = 0; x < DP / 16; ++x) {
    if ((2 * x + h) * 8 < D) {
      const X8 k = *reinterpret_cast<const X8*>(p + (2 * x + h) * 16);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s = __builtin_fmaf(static_cast<float>(f[x][e]), static_cast<float>(k[e]), s);
    }
    asm volatile("" ::: "memory");  // a piece at a time: few registers
  }
  return s + other_half(s);
}

// acc = acc * f + w * (the row at p), in the columns of a transposed result.
template <typename T, int DP>
__device__ __forceinline__ void add_row(f32x16* acc, float f, float w, const char* p, int D, int h) {
  typedef T x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i / 4) + 4 * h;
      if (col >= D) continue;
      const x4 v = *reinterpret_cast<const x4*>(p + col * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[d][i + e] = acc[d][i + e] * f + w * static_cast<float>(v[e]);
      asm volatile("" ::: "memory");
    }
}

// Whether a value of this lane's is infinite or NaN.
template <int DP>
__device__ __forceinline__ bool not_finite(const f32x16* acc) {
  float any = 0.0f;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) any = __builtin_fmaf(acc[d][i], 0.0f, any);  // 0, or NaN
  return any != 0.0f;
}

// A wave's queries once more, key by key and only over the keys that each one
// sees.  The matrix product of a tile that a query sees in part multiplies the
// values it does not see by 0, and 0 times an infinity or NaN is NaN: a wave
// that ends with such an output takes this way, so that what a masked value
// holds never shows.  (Finite inputs never come here, in the backward as long as
// scores stay below 2^30: an fp32 lse no longer tells probabilities apart there.)
template <typename T, int DP, typename X8>
__device__ __forceinline__ void rows_key_by_key(const X8* qf, const char* kp, int64_t k_row,
                                                const char* vp, int64_t v_row, int D, float c2,
                                                int end, int mine, int h, f32x16* o, float* m_out,
                                                float* sum_out) {
  float m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
#pragma unroll 1
  for (int j = 0; j < end; ++j, kp += k_row, vp += v_row) {
    const float s = dot_row<DP>(qf, kp, D, h);
    if (j >= mine) continue;
    const float m2 = fmaxf(m, s), base = m2 == -INFINITY ? 0.0f : m2;
    const float f = exp2_hw((m - base) * c2), p = exp2_hw((s - base) * c2);
    m = m2;
    sum = sum * f + p;
    add_row<T, DP>(o, f, p, vp, D, h);
  }
  *m_out = m;
  *sum_out = sum;
}

// One block: four waves, 32 queries each, of one list and one head, or on short
// lists of two or four heads that share their keys (twice four waves with
// NS = 2: two groups take alternate tiles of keys, and join their sums through
// LDS at the end).  Tiles of 64 keys and values go to LDS, the next one while
// this one is worked on.  Per tile a wave computes K Q^T (a query per lane, so
// that its probabilities are the next product's operand as they stand), the
// running maximum m and sum of exp(s - m) of its queries in registers, and adds
// V^T P^T to its outputs; outputs and sum are multiplied by exp(m - m') only when
// a maximum has grown by more than 2^8 (until then exp(s - m) <= 2^8).
// Probabilities are rounded to the input type for the second product, whose
// matrix instruction takes no wider one; sums, maxima and outputs are fp32.
//
// Bound: long lists by the issue of the matrix products and of the softmax's
// vector instructions between them (2 lists of 8192, 16 heads of 128 over 4:
// 518 to 566 us, 1.0 PFLOP/s of the visible pairs, matrix pipes busy for half the cycles,
// no LDS conflicts, 0.3 TB/s); many short ones by latency: to a block's first
// tile it is 4 to 5 us (the list, then queries and keys), of a life of 8 to 16
// (64 lists of 0 to 1000, 8 heads of 64 over 2: 48 to 51 us, 1.6 TB/s; 256 lists of
// up to 512, 8 heads of 96: 41 us).  Hence four waves and two tiles in turn: 3 or
// 4 blocks a CU; three tiles, or one or two waves a block, were slower.
template <typename T, typename I, int DP, int NS>
__global__ void __launch_bounds__(kRowWaves * NS * 64, 2) fwd_kernel(const FwdArgs a) {
  using E = Elem<T>;
  using X8 = typename E::x8;
  using Ti = Tile<DP>;
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int kTileBytes = kBN * DP * 2;
  __shared__ __attribute__((aligned(1024))) char lds[NS * 4 * kTileBytes];  // K0 V0 K1 V1 per group

  int head;
  int turn;
  head_and_turn(blockIdx.x, a.H >> a.pack, &head, &turn);
  const I* qo = static_cast<const I*>(a.q_offsets);
  const I* ko = static_cast<const I*>(a.k_offsets);
  Found f;
  if (a.turns != nullptr) {
    if (!find_planned(a.turns, a.n_turns, turn, &f)) return;
  } else if (a.ranked) {
    if (!find_ranked<true>(qo, ko, a.B, a.Nq, a.Nk, kRowShift - a.pack, a.causal != 0, turn, &f)) return;
  } else {
    if (!find_list<true>(qo, ko, a.B, a.Nq, a.Nk, kRowShift - a.pack, turn, &f)) return;
  }
  const Span sq = f.own, sk = f.other;
  const int tile = f.tile;
  const int BM = kRowWaves * 32 >> a.pack;      // the tile's queries
  if (tile < 0 || tile * BM >= sq.len) return;  // (below 0: offsets that decrease)

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, l = lane & 31, h = lane >> 5;
  const int group = wave / kRowWaves;                   // of the key tiles j with j % NS == group
  const int per_head = kRowWaves >> a.pack, sub = wave % kRowWaves;  // waves
  head = (head << a.pack) + (sub >> (2 - a.pack));
  const int row0 = tile * BM + (sub & (per_head - 1)) * 32;  // the wave's first query in the list
  const int64_t q_base = sq.start + row0;
  const int rows = rows_left(sq.len, row0, 32);
  const int Lk = sk.len;
  const int shift = Lk - sq.len;  // query i sees keys 0 .. i + shift
  // Keys that a query of the block, and one of the wave, sees at most; keys that
  // every query of the wave sees.
  const int blk_end = a.causal ? min_of(tile * BM + BM, sq.len) + shift : Lk;
  const int wave_end = rows == 0 ? 0 : a.causal ? row0 + rows + shift : Lk;
  const int all_end = a.causal ? min_of(row0 + shift + 1, Lk) : Lk;
  const int tiles = blk_end > 0 ? (blk_end + kBN - 1) / kBN : 0;
  const int mine = a.causal ? min_of(row0 + l + shift + 1, Lk) : Lk;  // this lane's query sees

  // Queries: the B operand of K Q^T.
  X8 qf[KS];
  load_rows<X8, KS>(qf, a.q + q_base * a.q_row + head * a.q_head, rows, a.q_row, a.D, l, h);
  __builtin_amdgcn_sched_barrier(0);

  typename Ti::template Loader<kBN, kRowWaves * 64> lk, lv;
  lk.init(tid % (kRowWaves * 64), a.k_row, a.D / 8);
  lv.init(tid % (kRowWaves * 64), a.v_row, a.D / 8);
  const char* kp = a.k + int64_t{sk.start} * a.k_row + (head / a.G) * a.k_head;
  const char* vp = a.v + int64_t{sk.start} * a.v_row + (head / a.G) * a.v_head;
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x16{};
  float m = -INFINITY, sum = 0.0f;
  const float c2 = a.scale * kLog2e;

  const Places<DP> at(lane, 0);

  // The restrict pointers tell the compiler that the copies into the next
  // tiles' LDS do not meet this tile's reads (it would wait for them).
  auto load_tile = [&](int j, char* __restrict__ dst) __attribute__((always_inline)) {
    const int n = rows_left(Lk, j * kBN, kBN);
    lk.load(make_rsrc(kp + static_cast<int64_t>(j) * kBN * a.k_row,
                      span_bytes(n, a.k_row, a.D * 2)), dst, wave % kRowWaves);
    lv.load(make_rsrc(vp + static_cast<int64_t>(j) * kBN * a.v_row,
                      span_bytes(n, a.v_row, a.D * 2)),
            dst + kTileBytes, wave % kRowWaves);
  };
  auto work = [&](int j, const char* __restrict__ cur, uint32_t buf,
                  char* __restrict__ next) __attribute__((always_inline)) {
    if (j + NS < tiles) load_tile(j + NS, next);
    const int k0 = j * kBN;
    if (k0 >= wave_end) return;
    const uint32_t ra = opaque(at.row + buf);

    f32x16 s[2]{};
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
      for (int b = 0; b < 2; ++b)  // two chains of products, each the other's wait
        s[b] = E::mfma32(lds_read16<X8>(cur + 32 * b * Ti::kRow + Ti::step2(ra, x)), qf[x], s[b]);

    if (k0 + kBN > all_end) {  // the tile reaches past a query's last key
      const int last = mine - k0 - 4 * h;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i / 4) + i % 4 >= last) s[b][i] = -INFINITY;
    }

    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = fmaxf(top, other_half(top));
    if (__any((top - m) * c2 > 8.0f)) {
      const float m2 = fmaxf(m, top);
      const float r = m2 == -INFINITY ? 1.0f : exp2_hw((m - m2) * c2);
      sum *= r;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= r;
      m = m2;
    }
    const float mc = m == -INFINITY ? 0.0f : m * c2;

    X8 p[4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = exp2_hw(__builtin_fmaf(s[b][i], c2, -mc));
        sum += e;
        p[2 * b + i / 8][i % 8] = static_cast<T>(e);
      }

    const uint32_t t0 = opaque(at.tr + buf), t1 = Ti::next8(t0);
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const char* f = cur + kTileBytes + 16 * x * Ti::kRow;
        o[d] = E::mfma32(join<X8>(lds_read_tr(f + Ti::step4(t0, d)), lds_read_tr(f + Ti::step4(t1, d))),
                         p[x], o[d]);
      }
  };

  char* const mine_lds = lds + group * 4 * kTileBytes;
  if (group < tiles) load_tile(group, mine_lds);
  for (int j = group, t = 0; t < (tiles + NS - 1) / NS; j += NS, ++t) {
    wait_and_barrier<0>();
    work(j, mine_lds, (t & 1) * 2 * kTileBytes, mine_lds + ((t + 1) & 1) * 2 * kTileBytes);
  }

  sum += other_half(sum);
  if constexpr (NS == 2) {
    // The second group's maxima, sums and outputs: 16 DB + 2 floats a lane.
    static_assert(sizeof(lds) >= kRowWaves * 64 * (16 * DB + 2) * 4, "the join's room");
    float* room = reinterpret_cast<float*>(lds) + wave % kRowWaves * 64 * (16 * DB + 2) + lane;
    wait_and_barrier<0>();
    if (group == 1) {
      room[0] = m;
      room[64] = sum;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) room[(2 + 16 * d + i) * 64] = o[d][i];
    }
    wait_and_barrier<0>();
    if (group == 1) return;
    const float mb = room[0], top = fmaxf(m, mb);
    const float fa = top == -INFINITY ? 0.0f : exp2_hw((m - top) * c2);
    const float fb = top == -INFINITY ? 0.0f : exp2_hw((mb - top) * c2);
    sum = sum * fa + room[64] * fb;
    m = top;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * fa + room[(2 + 16 * d + i) * 64] * fb;
  }
  if (__builtin_expect(a.causal && __any(l < rows && not_finite<DP>(o)), 0))
    rows_key_by_key<T, DP>(qf, kp, a.k_row, vp, a.v_row, a.D, c2, wave_end, mine, h, o, &m, &sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  store_rows<T, DP>(static_cast<T*>(a.out) + (q_base * a.H + head) * a.D, o, inv, rows, a.H, a.D, l, h);
  if (a.lse != nullptr && h == 0 && l < rows)
    a.lse[int64_t{head} * a.Nq + q_base + l] = sum == 0.0f ? -INFINITY : m * a.scale + __logf(sum);
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// With delta_i = dO_i.o_i and dP_ij = dO_i.v_j:
//   dS_ij = p_ij (dP_ij - delta_i),
//   dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i p_ij dO_i,
// the last two also over the query heads that share the key-value head.  Two
// launches, each of which owns what it writes (no atomics: the same bits every
// time): the first has the queries' tiles and leaves each query's delta and
// base-2 lse for the second, which has the keys' tiles.  Scores are computed
// in both, seven products where five would do, which is less than what summing
// dQ over key tiles through memory costs.

// dS goes into a matrix product in the input type, and fp16 ends at 65504, which
// finite gradients' dS can pass (dO of 5e3 and v of 4 in 128 columns give dP of
// 2e5; scale, and small q and k, may bring the gradients back into range).  So for
// fp16 a column (a query of the first launch, a key of the second) of 32 rows of dS
// is looked at before its rounding, and where one passes the range the column's
// dS is multiplied from there on by a power of two that brings it below 2^15, and
// what has been summed of it by the same: exact, until the caller divides the sums
// by it.  Such a factor f leaves dS with 11 bits down to 2^-14 / f, which is 2^-28
// of the column's largest or less.  It waits in LDS (`mine`, of this lane): in the
// ordinary case, fitted == false, only the maxima of |dS| and a vote are spent (4
// lists of 4096, 16 heads of 128 over 4, fp16: backward 1024 -> 1040 us; 64 of 0 to
// 1000, 8 of 64 over 2: 184 -> 189; one of 1024, 8 of 128: 65, and 73 where columns
// need factors).
// Returns whether the wave's columns have factors.
template <int DB>
__device__ __forceinline__ bool fit_range(f32x16& ds, f32x16* acc, float* mine, bool fitted) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
  if (__builtin_expect(!fitted && !__any(top > 65504.0f), 1)) return false;
  const float before = fitted ? *mine : 1.0f;
  float f = before;
  top = fmaxf(top, other_half(top));  // the column's other 16 rows
  // An infinity is one of the inputs' and stays one.
  if (top * f > 65504.0f && top < INFINITY) f = __builtin_ldexpf(1.0f, 15 - __builtin_amdgcn_frexp_expf(top));
  const float r = f / before;
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] *= r;
  ds *= f;
  *mine = f;
  return true;
}

struct BwdArgs {
  const char *q, *k, *v, *out, *grad;  // bytes; out and grad with q's shape
  uint32_t q_row, k_row, v_row, o_row, g_row;
  int64_t q_head, k_head, v_head, o_head, g_head;
  const void *q_offsets, *k_offsets;
  int32_t B, Nq, Nk;
  int32_t H, Hkv, G, D;
  int32_t causal;
  int32_t pack;                    // log2 of the heads of a block (queries' launch)
  int32_t ranked;                  // find_ranked finds the tiles
  const Turn *q_turns, *k_turns;   // find_planned does, if not null
  int32_t n_q_turns, n_k_turns;
  float scale;
  const float* lse;                    // [H, Nq]
  float *lse2, *delta;                 // [H, Nq], workspace
  void *dq, *dk, *dv;                  // contiguous
  int32_t shares;                      // of a key tile's queries (bwd_kv_kernel)
  float* sums;                         // [shares, 2, Nk, Hkv, D], workspace if shares > 1
};

// The queries' launch: tiles as in the forward.  A wave keeps Q and dO of its 32
// queries as operands and dQ as sums; per tile it computes S and dP with a query
// per lane and adds K^T dS^T.  Where all keys of a query fit one tile, delta is
// sum_j p_ij dP_ij from there (exact to the rounding of P) and the output is not
// read; else it is dO.o.  Bound as the forward's (4 lists of 4096, 16 heads of 128
// over 4: 409 us, 1.0 PFLOP/s, matrix pipes 53%; 256 lists of up to 512, 8 heads
// of 96: 50 us).
template <typename T, typename I, int DP, int NS>
__global__ void __launch_bounds__(kRowWaves * NS * 64, DP <= 64 ? 4 : NS == 1 && DP == 96 ? 3 : 2) bwd_q_kernel(const BwdArgs a) {
  using E = Elem<T>;
  using X8 = typename E::x8;
  using Ti = Tile<DP>;
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int kTileBytes = kBN * DP * 2;
  __shared__ __attribute__((aligned(1024))) char lds[NS * 4 * kTileBytes + (E::kNarrow ? kRowWaves * NS * 64 * 4 : 0)];

  int head;
  int turn;
  head_and_turn(blockIdx.x, a.H >> a.pack, &head, &turn);
  const I* qo = static_cast<const I*>(a.q_offsets);
  const I* ko = static_cast<const I*>(a.k_offsets);
  Found f;
  if (a.q_turns != nullptr) {
    if (!find_planned(a.q_turns, a.n_q_turns, turn, &f)) return;
  } else if (a.ranked) {
    if (!find_ranked<true>(qo, ko, a.B, a.Nq, a.Nk, kRowShift - a.pack, a.causal != 0, turn, &f)) return;
  } else {
    if (!find_list<true>(qo, ko, a.B, a.Nq, a.Nk, kRowShift - a.pack, turn, &f)) return;
  }
  const Span sq = f.own, sk = f.other;
  const int tile = f.tile;
  const int BM = kRowWaves * 32 >> a.pack;      // the tile's queries
  if (tile < 0 || tile * BM >= sq.len) return;  // (below 0: offsets that decrease)

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, l = lane & 31, h = lane >> 5;
  const int group = wave / kRowWaves;                   // of the key tiles j with j % NS == group
  const int per_head = kRowWaves >> a.pack, sub = wave % kRowWaves;  // waves
  head = (head << a.pack) + (sub >> (2 - a.pack));
  const int row0 = tile * BM + (sub & (per_head - 1)) * 32;  // the wave's first query in the list
  const int64_t q_base = sq.start + row0;
  const int rows = rows_left(sq.len, row0, 32);
  const int Lk = sk.len;
  const int shift = Lk - sq.len;  // query i sees keys 0 .. i + shift
  // Keys that a query of the block, and one of the wave, sees at most; keys that
  // every query of the wave sees.
  const int blk_end = a.causal ? min_of(tile * BM + BM, sq.len) + shift : Lk;
  const int wave_end = rows == 0 ? 0 : a.causal ? row0 + rows + shift : Lk;
  const int all_end = a.causal ? min_of(row0 + shift + 1, Lk) : Lk;
  const int tiles = blk_end > 0 ? (blk_end + kBN - 1) / kBN : 0;
  const int mine = a.causal ? min_of(row0 + l + shift + 1, Lk) : Lk;  // this lane's query sees

  X8 qf[KS], gf[KS];
  load_rows<X8, KS>(qf, a.q + q_base * a.q_row + head * a.q_head, rows, a.q_row, a.D, l, h);
  load_rows<X8, KS>(gf, a.grad + q_base * a.g_row + head * a.g_head, rows, a.g_row, a.D, l, h);
  float delta = 0.0f, lse2 = 0.0f;
  if (wave_end > kBN) {  // else delta comes from the first tile
    X8 of[KS];
    load_rows<X8, KS>(of, a.out + q_base * a.o_row + head * a.o_head, rows, a.o_row, a.D, l, h);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta = __builtin_fmaf(static_cast<float>(of[s][e]), static_cast<float>(gf[s][e]), delta);
    delta += other_half(delta);
  }
  if (l < rows) {
    const int64_t at = int64_t{head} * a.Nq + q_base + l;
    lse2 = a.lse[at] * kLog2e;
    if (h == 0 && group == 0) {
      a.lse2[at] = lse2;
      a.delta[at] = delta;
    }
  }

  typename Ti::template Loader<kBN, kRowWaves * 64> lk, lv;
  lk.init(tid % (kRowWaves * 64), a.k_row, a.D / 8);
  lv.init(tid % (kRowWaves * 64), a.v_row, a.D / 8);
  const char* kp = a.k + int64_t{sk.start} * a.k_row + (head / a.G) * a.k_head;
  const char* vp = a.v + int64_t{sk.start} * a.v_row + (head / a.G) * a.v_head;

  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = f32x16{};
  bool fitted = false;  // fit_range, and where this lane's factor is
  auto factor = [&] { return reinterpret_cast<float*>(lds + NS * 4 * kTileBytes) + wave * 64 + lane_again(); };
  const float c2 = a.scale * kLog2e;
  const Places<DP> at(lane, 0);

  auto load_tile = [&](int j, char* __restrict__ dst) __attribute__((always_inline)) {
    const int n = rows_left(Lk, j * kBN, kBN);
    lk.load(make_rsrc(kp + static_cast<int64_t>(j) * kBN * a.k_row,
                      span_bytes(n, a.k_row, a.D * 2)), dst, wave % kRowWaves);
    lv.load(make_rsrc(vp + static_cast<int64_t>(j) * kBN * a.v_row,
                      span_bytes(n, a.v_row, a.D * 2)),
            dst + kTileBytes, wave % kRowWaves);
  };
  auto work = [&](int j, const char* __restrict__ cur, uint32_t buf,
                  char* __restrict__ next) __attribute__((always_inline)) {
    if (j + NS < tiles) load_tile(j + NS, next);
    if (j == 0 && wave_end <= kBN) {
      // These queries see no key past this tile: delta = sum_j p_ij dP_ij in fp32
      // comes from the tile itself, at the price of its scores once more.  From
      // the rounded output it is off by that rounding, which shows most where few
      // keys share a large gradient (256 lists of up to 512: dQ's error against
      // 64 bits 2.6e-3 -> 2.4e-3, its largest halved).
      float sum = 0.0f;
#pragma unroll 1
      for (int k0 = 0; k0 < wave_end; k0 += 32) {
        const uint32_t ra = opaque(at.row + buf + k0 * Ti::kRow);
        f32x16 s{}, dp{};
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          s = E::mfma32(lds_read16<X8>(cur + Ti::step2(ra, x)), qf[x], s);
          dp = E::mfma32(lds_read16<X8>(cur + kTileBytes + Ti::step2(ra, x)), gf[x], dp);
        }
        const int last = mine - k0 - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float w = exp2_hw(__builtin_fmaf(s[i], c2, -lse2)) * dp[i];
          sum += 8 * (i / 4) + i % 4 >= last ? 0.0f : w;
        }
      }
      delta = sum + other_half(sum);
      if (h == 0 && l < rows) a.delta[int64_t{head} * a.Nq + q_base + l] = delta;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int k0 = j * kBN + 32 * b;
      if (k0 >= wave_end) return;
      const uint32_t ra = opaque(at.row + buf), t0 = opaque(at.tr + buf), t1 = Ti::next8(t0);
      const char* kt = cur + 32 * b * Ti::kRow;
      const char* vt = kt + kTileBytes;
      f32x16 s{}, dp{};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        s = E::mfma32(lds_read16<X8>(kt + Ti::step2(ra, x)), qf[x], s);
        dp = E::mfma32(lds_read16<X8>(vt + Ti::step2(ra, x)), gf[x], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = exp2_hw(__builtin_fmaf(s[i], c2, -lse2)) * (dp[i] - delta);
      if (k0 + 32 > all_end) {
        const int last = mine - k0 - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 >= last) s[i] = 0.0f;
      }
      if constexpr (E::kNarrow) fitted = fit_range<DB>(s, dq, factor(), fitted);
      X8 ds[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i / 8][i % 8] = static_cast<T>(s[i]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const char* f = kt + 16 * x * Ti::kRow;
          dq[d] = E::mfma32(join<X8>(lds_read_tr(f + Ti::step4(t0, d)), lds_read_tr(f + Ti::step4(t1, d))),
                            ds[x], dq[d]);
        }
    }
  };

  char* const mine_lds = lds + group * 4 * kTileBytes;
  if (group < tiles) load_tile(group, mine_lds);
  for (int j = group, t = 0; t < (tiles + NS - 1) / NS; j += NS, ++t) {
    wait_and_barrier<0>();
    work(j, mine_lds, (t & 1) * 2 * kTileBytes, mine_lds + ((t + 1) & 1) * 2 * kTileBytes);
  }
  if (E::kNarrow && fitted) {
    const float inv = 1.0f / *factor();
#pragma unroll
    for (int d = 0; d < DB; ++d) dq[d] *= inv;
  }

  if constexpr (NS == 2) {
    static_assert(NS * 4 * kTileBytes >= kRowWaves * 64 * 16 * DB * 4, "the join's room");
    float* room = reinterpret_cast<float*>(lds) + wave % kRowWaves * 64 * 16 * DB + lane;
    wait_and_barrier<0>();
    if (group == 1) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) room[(16 * d + i) * 64] = dq[d][i];
    }
    wait_and_barrier<0>();
    if (group == 1) return;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dq[d][i] += room[(16 * d + i) * 64];
  }
  if (__builtin_expect(a.causal && __any(l < rows && not_finite<DP>(dq)), 0)) {
    // As in the forward: keys that a query does not see leave the products.  (The
    // rows again, for registers' sake.)
    X8 qr[KS], gr[KS];
    load_rows<X8, KS>(qr, a.q + q_base * a.q_row + head * a.q_head, rows, a.q_row, a.D, l, h);
    load_rows<X8, KS>(gr, a.grad + q_base * a.g_row + head * a.g_head, rows, a.g_row, a.D, l, h);
#pragma unroll
    for (int d = 0; d < DB; ++d) dq[d] = f32x16{};
#pragma unroll 1
    for (int j = 0; j < wave_end; ++j, kp += a.k_row, vp += a.v_row) {
      const float s = dot_row<DP>(qr, kp, a.D, h), dp = dot_row<DP>(gr, vp, a.D, h);
      if (j < mine)
        add_row<T, DP>(dq, 1.0f, exp2_hw(__builtin_fmaf(s, c2, -lse2)) * (dp - delta), kp, a.D, h);
    }
  }
  store_rows<T, DP>(static_cast<T*>(a.dq) + (q_base * a.H + head) * a.D, dq, a.scale, rows, a.H, a.D, l, h);
}

// The keys' launch: a wave owns 32 keys and their sums over every query head of
// the group and every query that sees them (half of them with NQ = 2: two
// groups of waves take alternate 64-query blocks and join their sums through
// LDS at the end).  Queries and dO go through LDS with their lse and delta;
// scores come out with a key per lane.  D = 128 takes 192 registers for K, V,
// dK and dV: scores are used up before dP is computed, which leaves two waves
// per SIMD.  Bound: the matrix products' issue and the LDS reads that feed them
// with only two waves to hide either (4 lists of 4096, 16 heads of 128 over 4:
// 610 us, 0.9 PFLOP/s, matrix pipes 44%); short lists by latency as above (256
// lists of up to 512, 8 heads of 96: 63 us).
template <typename T, typename I, int DP, int NQ>
__global__ void __launch_bounds__(kRowWaves * NQ * 64, 2) bwd_kv_kernel(const BwdArgs a) {
  using E = Elem<T>;
  using X8 = typename E::x8;
  using Ti = Tile<DP>;
  constexpr int KS = DP / 16, DB = DP / 32, BM = kRowWaves * 32, BQ = 64 * NQ, THREADS = kRowWaves * NQ * 64;
  constexpr int kTileBytes = BQ * DP * 2;
  constexpr int kStat = BQ * 4;
  constexpr int kBuf = 2 * kTileBytes + 2 * kStat;  // Q, dO, lse2, delta
  // The last piece of V waits in LDS where the registers run out: a spilled one
  // is loaded from memory, and its wait is one for the tiles in flight too (4 x
  // 4096, 16 heads of 128: backward 1047 -> 1021 us).
  constexpr bool kKeep = DP == 128 && NQ == 2;
  constexpr int kInRegs = kKeep ? KS - 1 : KS;
  constexpr int kFactors = 2 * kBuf + (kKeep ? THREADS * 16 : 0);
  __shared__ __attribute__((aligned(1024))) char lds[kFactors + (E::kNarrow ? THREADS * 4 : 0)];
  static_assert(NQ == 1 || 2 * kBuf >= BM * DP * 4, "the join's room");

  int kvh;
  int turn;
  head_and_turn(blockIdx.x, a.Hkv, &kvh, &turn);
  const I* qo = static_cast<const I*>(a.q_offsets);
  const I* ko = static_cast<const I*>(a.k_offsets);
  Found f;
  if (a.k_turns != nullptr) {
    if (!find_planned(a.k_turns, a.n_k_turns, turn, &f)) return;
  } else if (a.ranked) {
    if (!find_ranked<false>(ko, qo, a.B, a.Nk, a.Nq, kRowShift, a.causal != 0, turn, &f)) return;
  } else {
    if (!find_list<false>(ko, qo, a.B, a.Nk, a.Nq, kRowShift, turn, &f)) return;
  }
  const Span sk = f.own, sq = f.other;
  const int tile = f.tile;
  if (tile < 0 || tile * BM >= sk.len) return;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wave / kRowWaves;  // which 64 of a tile's queries
  const int lane = tid & 63, l = lane & 31, h = lane >> 5;
  const int key0 = tile * BM + wave % kRowWaves * 32;
  const int64_t k_base = sk.start + key0;
  const int keys = rows_left(sk.len, key0, 32);
  const int Lq = sq.len;
  const int shift = sk.len - Lq;
  // From the first query that sees a key of the block, to a whole 64.
  const int first = a.causal && tile * BM > shift ? (tile * BM - shift) / 64 * 64 : 0;
  const int per = Lq > first ? (Lq - first + BQ - 1) / BQ : 0;
  // This share's blocks of BQ queries, counted through the group's heads.
  const int share = blockIdx.y;
  const int begin = static_cast<int>(int64_t{per} * a.G * share / a.shares);
  const int end = static_cast<int>(int64_t{per} * a.G * (share + 1) / a.shares);

  X8 kf[KS], vf[KS];
  load_rows<X8, KS>(kf, a.k + k_base * a.k_row + kvh * a.k_head, keys, a.k_row, a.D, l, h);
  load_rows<X8, KS>(vf, a.v + k_base * a.v_row + kvh * a.v_head, keys, a.v_row, a.D, l, h);
  if constexpr (kKeep) *reinterpret_cast<X8*>(lds + 2 * kBuf + tid * 16) = vf[KS - 1];

  typename Ti::template Loader<BQ, THREADS> lq, lg;
  lq.init(tid, a.q_row, a.D / 8);
  lg.init(tid, a.g_row, a.D / 8);
  const int64_t qs = sq.start;

  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = f32x16{};
  bool fitted = false;  // fit_range, and where this lane's factor is
  auto factor = [&] { return reinterpret_cast<float*>(lds + kFactors) + wave * 64 + lane_again(); };
  const float c2 = a.scale * kLog2e;
  const Places<DP> at(lane, 64 * part);

  auto load_tile = [&](int g, int t, char* __restrict__ dst) __attribute__((always_inline)) {
    const int head = kvh * a.G + g;
    const int i0 = first + t * BQ;
    const int n = rows_left(Lq, i0, BQ);
    lq.load(make_rsrc(a.q + (qs + i0) * a.q_row + head * a.q_head,
                      span_bytes(n, a.q_row, a.D * 2)), dst, wave);
    lg.load(make_rsrc(a.grad + (qs + i0) * a.g_row + head * a.g_head,
                      span_bytes(n, a.g_row, a.D * 2)),
            dst + kTileBytes, wave);
    const int64_t s0 = int64_t{head} * a.Nq + qs + i0;
    if (wave < 2 * NQ) {  // 64 values each
      const float* from = (wave < NQ ? a.lse2 : a.delta) + s0;
      load4_to_lds(make_rsrc(from, n * 4), dst + 2 * kTileBytes + wave * 256,
                   (wave % NQ * 64 + lane_again()) * 4);
    }
  };
  auto work = [&](int t, const char* __restrict__ cur, uint32_t buf, char* __restrict__ next, int gn,
                  int tn, bool more) __attribute__((always_inline)) {
    if (more) load_tile(gn, tn, next);
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
      const int i0 = first + t * BQ + 64 * part + 32 * b;
      if (keys == 0 || i0 >= Lq) return;
      if (a.causal && key0 > i0 + 31 + shift) continue;
      const uint32_t from32 = buf + 32 * b * Ti::kRow;
      const uint32_t ra = opaque(at.row + from32), t0 = opaque(at.tr + from32), t1 = Ti::next8(t0);
      const char* gt = cur + kTileBytes;
      const int lc = lane_again() & 31, h4 = lane_again() >> 5 << 2;
      const char* st = cur + buf + 2 * kTileBytes + (64 * part + 32 * b + h4) * 4;
      f32x16 s{}, dp{};
#pragma unroll
      for (int x = 0; x < KS; ++x) s = E::mfma32(lds_read16<X8>(cur + Ti::step2(ra, x)), kf[x], s);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(st + 32 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[4 * u + e] = exp2_hw(__builtin_fmaf(s[4 * u + e], c2, -ls[e]));
      }
      // Query i0 + r sees key0 + l if r >= key0 + l - shift - i0.
      const bool masked = a.causal && key0 + 31 > i0 + shift;
      const int from = key0 + lc - shift - i0 - h4;
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 < from) s[i] = 0.0f;
      }
      X8 p[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i / 8][i % 8] = static_cast<T>(s[i]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const char* f = gt + 16 * x * Ti::kRow;
          dv[d] = E::mfma32(join<X8>(lds_read_tr(f + Ti::step4(t0, d)), lds_read_tr(f + Ti::step4(t1, d))),
                            p[x], dv[d]);
        }
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t rb = opaque(at.row + from32);
#pragma unroll
      for (int x = 0; x < kInRegs; ++x) dp = E::mfma32(lds_read16<X8>(gt + Ti::step2(rb, x)), vf[x], dp);
      if constexpr (kKeep)
        dp = E::mfma32(lds_read16<X8>(gt + Ti::step2(rb, KS - 1)),
                       lds_read16<X8>(cur + 2 * kBuf + (wave * 64 + lane_again()) * 16), dp);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 de = *reinterpret_cast<const f32x4*>(st + kStat + 32 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * u + e] = s[4 * u + e] * (dp[4 * u + e] - de[e]);
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 < from) dp[i] = 0.0f;
      }
      if constexpr (E::kNarrow) fitted = fit_range<DB>(dp, dk, factor(), fitted);
      X8 ds[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i / 8][i % 8] = static_cast<T>(dp[i]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const char* f = cur + 16 * x * Ti::kRow;
          dk[d] = E::mfma32(join<X8>(lds_read_tr(f + Ti::step4(t0, d)), lds_read_tr(f + Ti::step4(t1, d))),
                            ds[x], dk[d]);
        }
    }
  };

  uint32_t buf = 0;
  if (begin < end) {
    int g = begin / per, t = begin - g * per;
    load_tile(g, t, lds);
    for (int left = end - begin; left > 0; --left, buf = kBuf - buf) {
      const int tn = t + 1 < per ? t + 1 : 0, gn = t + 1 < per ? g : g + 1;
      wait_and_barrier<0>();
      work(t, lds, buf, lds + (kBuf - buf), gn, tn, left > 1);
      t = tn;
      g = gn;
    }
  }
  if (E::kNarrow && fitted) {
    const float inv = 1.0f / *factor();
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] *= inv;
  }

  if constexpr (NQ == 2) {
    // One lane's values of a block of columns: 16 x 64 floats per step.
    float* room = reinterpret_cast<float*>(lds) + wave % kRowWaves * 32 * DP + lane;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      f32x16* x = pass == 0 ? dk : dv;
      __syncthreads();
      if (part == 1) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) room[(d * 16 + i) * 64] = x[d][i];
      }
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[d][i] += room[(d * 16 + i) * 64];
      }
    }
    if (part == 1) return;
  }
  // Counted anew: they would take registers through the loop.
  const int le = lane_again() & 31, he = lane_again() >> 5;
  if (__builtin_expect(a.causal && __any(le < keys && (not_finite<DP>(dk) || not_finite<DP>(dv))), 0)) {
    // As in the forward: queries that do not see a key leave its products.  (The
    // rows again, for registers' sake.)
    X8 kr[KS], vr[KS];
    load_rows<X8, KS>(kr, a.k + k_base * a.k_row + kvh * a.k_head, keys, a.k_row, a.D, le, he);
    load_rows<X8, KS>(vr, a.v + k_base * a.v_row + kvh * a.v_head, keys, a.v_row, a.D, le, he);
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = f32x16{};
#pragma unroll 1
    for (int u = begin; u < end; ++u) {
      const int head = kvh * a.G + u / per;
      const int i0 = first + u % per * BQ, i1 = min_of(i0 + BQ, Lq);
#pragma unroll 1
      for (int i = i0; i < i1; ++i) {
        const char* qp = a.q + (qs + i) * a.q_row + head * a.q_head;
        const char* gp = a.grad + (qs + i) * a.g_row + head * a.g_head;
        const int64_t at_i = int64_t{head} * a.Nq + qs + i;
        const float s = dot_row<DP>(kr, qp, a.D, he);
        __builtin_amdgcn_sched_barrier(0);
        const float dp = dot_row<DP>(vr, gp, a.D, he);
        __builtin_amdgcn_sched_barrier(0);
        if (key0 + le > i + shift) continue;
        const float p = exp2_hw(__builtin_fmaf(s, c2, -a.lse2[at_i]));
        add_row<T, DP>(dv, 1.0f, p, gp, a.D, he);
        __builtin_amdgcn_sched_barrier(0);
        add_row<T, DP>(dk, 1.0f, p * (dp - a.delta[at_i]), qp, a.D, he);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  const int64_t to = (k_base * a.Hkv + kvh) * a.D;
  if (a.shares > 1) {
    const int64_t all = int64_t{a.Nk} * a.Hkv * a.D;
    store_sums<DP>(a.sums + 2 * share * all + to, dk, keys, a.Hkv, a.D, le, he);
    store_sums<DP>(a.sums + (2 * share + 1) * all + to, dv, keys, a.Hkv, a.D, le, he);
    return;
  }
  store_rows<T, DP>(static_cast<T*>(a.dk) + to, dk, a.scale, keys, a.Hkv, a.D, le, he);
  store_rows<T, DP>(static_cast<T*>(a.dv) + to, dv, 1.0f, keys, a.Hkv, a.D, le, he);
}

// dK and dV from their shares' sums, added in the shares' order, four values a
// thread.  Bound: reading the sums, which the caches still hold.
template <typename T>
__global__ void __launch_bounds__(256) join_shares_kernel(const BwdArgs a) {
  typedef T x4 __attribute__((ext_vector_type(4)));
  const int64_t all = int64_t{a.Nk} * a.Hkv * a.D;
  const int64_t i = (int64_t{blockIdx.x} * 256 + threadIdx.x) * 4;
  if (i >= all) return;
  const bool v = blockIdx.y == 1;
  const float* p = a.sums + (v ? all : 0) + i;
  f32x4 sum{};
#pragma unroll 4
  for (int s = 0; s < a.shares; ++s) sum += *reinterpret_cast<const f32x4*>(p + 2 * s * all);
  const float scale = v ? 1.0f : a.scale;
  x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(sum[e] * scale);
  *reinterpret_cast<x4*>(static_cast<T*>(v ? a.dv : a.dk) + i) = w;
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------

// Waves beyond a block's four where the launch's tiles of 128 rows do not fill
// the chip, on lists long enough to share out.  Times in us:
//   key tiles over two groups, forward: 1 list of 4096, 8 heads of 128 (256 tiles)
//   94 -> 78; 16 lists of 128 queries and 1128 keys, 8 of 128, 34.4 -> 32.5; 1 of
//   5282, 8 of 64 (336 tiles) 84 -> 67; 2 of 4096 (512 tiles) 82 -> 73, 8 of 128
//   121 -> 94; 4 of 2048 (512 tiles) 45.2 -> 41.6, 8 of 128 65.6 -> 68.3; 8 of 1024
//   (512 tiles), 8 of 128, 38.6 -> 48.4;
//   backward's keys, queries over two groups (whole backward), 8 heads of 128: 1 x
//   4096 310 -> 258, 4 x 2048 (512 tiles) 184 -> 173, 6 x 2048 211 -> 233, 16 x 512
//   (512 tiles) 71 -> 81, the same with 2 key-value heads 127 -> 101.
bool split_keys(int64_t Nq, int64_t Nk, int64_t B, int64_t H) {
  if (B == 0) return false;
  const int64_t tiles = ceil_div(Nq, 128) * H, mean = Nk / B, cus = num_cus();
  return (2 * tiles <= 3 * cus && mean >= 512) || (tiles <= 2 * cus && mean >= 4096);
}
bool split_queries(int64_t Nq, int64_t Nk, int64_t B, int64_t Hkv, int64_t G) {
  return B > 0 && ceil_div(Nk, 128) * Hkv <= 2 * num_cus() && Nq / B * G >= 1024;
}

// Shares of a key tile's queries where the tiles leave part of the chip idle, joined
// by a third launch: up to two blocks of four waves, or one of eight, for every CU,
// and two tiles of queries in each share of a list of mean length.  Whole
// backward in us, without and with them (more than 4, 8 or 16 shares once the chip
// is full gain no more): one list of 1059, 8 heads of 128 over 1: 291 -> 74; 4096,
// 8 of 64 over 1: 632 -> 154; 4096, 16 of 128 over 2: 1026 -> 404; 2 of 400, 8 of
// 64 over 1: 86 -> 35; 4 of 1 to 1000, 4 heads of 96: 70 -> 60; 2 of 300, 2 heads
// of 128: 42 -> 39; with four tiles a share at least 8 of 1 to 500, 8 of 64 over 1,
// 52, with two 42, with one 44.
int32_t query_shares(const mx_attention_problem* p) {
  if (p->B == 0 || p->Nk == 0) return 1;
  const int64_t G = p->H / p->Hkv, blocks = ceil_div(p->Nk, 128) * p->Hkv;
  const bool two = split_queries(p->Nq, p->Nk, p->B, p->Hkv, G);
  const int64_t room = (two ? 1 : 2) * static_cast<int64_t>(num_cus()) / blocks;
  const int64_t work = p->Nq / p->B * G / (two ? 256 : 128);
  const int64_t n = std::min<int64_t>({room, work, 16});

  return n > 1 ? static_cast<int32_t>(n) : 1;
}

// Query heads (log2) that a block of the queries' launches takes, of those that
// share a key-value head: its four waves have 32 queries of four heads, 64 of two
// or 128 of one, and read the same keys.  Short lists leave fewer waves without a
// query; long ones start more blocks that must find their tile.  In us, one head
// and as many as there are: 117 lists of 27 with 249 keys, 16 heads of 128 over 4:
// forward 32.5 -> 21.8, with the backward 114 -> 87; 200 of 1 to 60, 8 of 64 over
// 2: 12.4 -> 9.0; 173 of 1 to 344, 4 of 80 over 1, with the backward 116 -> 105; 32
// of 1 to 600, 8 of 96 over 4: 22.6 -> 21.8; 64 of 1 to 1000, 8 of 64 over 2: 48.5
// -> 49.4; 16 of 512, 8 of 128 over 2: 23.0 -> 24.7; 2 of 8192: the same.
int heads_packed(const mx_attention_problem* p) {
  const int32_t G = p->H / p->Hkv;
  if (p->Nq > 384 * p->B) return 0;
  return G % 4 == 0 ? 2 : G % 2 == 0 ? 1 : 0;
}

int blocks_of(int64_t rows, int64_t B, int64_t heads, int pack, unsigned* blocks) {
  const int64_t n = tile_turns(rows, B, 128 >> pack) * (heads >> pack);
  MX_REQUIRE(n < (1ll << 23), "too many tiles: %lld", (long long)n);  // of 512 threads in 32 bits
  *blocks = static_cast<unsigned>(n);
  return MX_OK;
}

template <typename T, typename I, int DP>
int launch_fwd(const FwdArgs& a, hipStream_t stream) {
  unsigned blocks;
  if (int rc = blocks_of(a.Nq, a.B, a.H, a.pack, &blocks)) return rc;
  if (split_keys(a.Nq, a.Nk, a.B, a.H))
    fwd_kernel<T, I, DP, 2><<<dim3(blocks), 512, 0, stream>>>(a);
  else
    fwd_kernel<T, I, DP, 1><<<dim3(blocks), 256, 0, stream>>>(a);
  MX_LAUNCH_CHECK();
  return MX_OK;
}

template <typename T, typename I, int DP>
int launch_bwd(const BwdArgs& a, hipStream_t stream) {
  unsigned qblocks, kblocks;
  if (int rc = blocks_of(a.Nq, a.B, a.H, a.pack, &qblocks)) return rc;
  if (int rc = blocks_of(a.Nk, a.B, a.Hkv, 0, &kblocks)) return rc;
  if (a.Nq > 0) {
    if (split_keys(a.Nq, a.Nk, a.B, a.H))
      bwd_q_kernel<T, I, DP, 2><<<dim3(qblocks), 512, 0, stream>>>(a);
    else
      bwd_q_kernel<T, I, DP, 1><<<dim3(qblocks), 256, 0, stream>>>(a);
  }
  if (a.Nk > 0 && a.dk != nullptr) {
    const dim3 grid(kblocks, a.shares);
    if (split_queries(a.Nq, a.Nk, a.B, a.Hkv, a.G))
      bwd_kv_kernel<T, I, DP, 2><<<grid, 512, 0, stream>>>(a);
    else
      bwd_kv_kernel<T, I, DP, 1><<<grid, 256, 0, stream>>>(a);
    if (a.shares > 1) {
      const int64_t n = ceil_div(int64_t{a.Nk} * a.Hkv * a.D, 1024);
      join_shares_kernel<T><<<dim3(static_cast<unsigned>(n), 2), 256, 0, stream>>>(a);
    }
  }
  MX_LAUNCH_CHECK();
  return MX_OK;
}

// The instance of a call: element type, index type, and the head width rounded
// up to 32 (zeros fill the rest of a tile's rows).
#define MX_ATTN_DISPATCH(LAUNCH, T, args, index_bytes, stream)                          \
  (index_bytes == 8 ? ((args).D <= 32   ? LAUNCH<T, int64_t, 32>(args, stream)          \
                       : (args).D <= 64 ? LAUNCH<T, int64_t, 64>(args, stream)          \
                       : (args).D <= 96 ? LAUNCH<T, int64_t, 96>(args, stream)          \
                                        : LAUNCH<T, int64_t, 128>(args, stream))        \
                    : ((args).D <= 32   ? LAUNCH<T, int32_t, 32>(args, stream)          \
                       : (args).D <= 64 ? LAUNCH<T, int32_t, 64>(args, stream)          \
                       : (args).D <= 96 ? LAUNCH<T, int32_t, 96>(args, stream)          \
                                        : LAUNCH<T, int32_t, 128>(args, stream)))

// One strided [N, heads, D] operand: its strides in bytes, checked for what
// the kernels assume (16-byte rows; 64 rows of a tile within a descriptor).
int check_operand(const char* name, const mx_attention_tensor* t, int32_t D, int64_t N) {
  MX_REQUIRE(t != nullptr && (N == 0 || t->data != nullptr), "%s is null", name);
  MX_REQUIRE(reinterpret_cast<uintptr_t>(t->data) % 16 == 0 && t->row_stride % 8 == 0 &&
                 t->head_stride % 8 == 0,
             "%s: rows and heads must start at multiples of 16 bytes", name);
  MX_REQUIRE(t->row_stride >= D || N <= 1, "%s: row stride %lld below D = %d", name,
             (long long)t->row_stride, D);
  MX_REQUIRE(t->row_stride >= 0 && t->row_stride <= (1ll << 23), "%s: row stride %lld above 2^23 elements", name,
             (long long)t->row_stride);
  MX_REQUIRE(t->head_stride >= 0, "%s: negative head stride", name);
  return MX_OK;
}

uint32_t row_bytes(const mx_attention_tensor* t) { return static_cast<uint32_t>(t->row_stride * 2); }

int check_problem(const mx_attention_problem* p) {
  MX_REQUIRE(p != nullptr, "problem is null");
  MX_REQUIRE(p->dtype == MX_DTYPE_F16 || p->dtype == MX_DTYPE_BF16, "dtype %d is not fp16 or bf16", p->dtype);
  MX_REQUIRE(p->index_bytes == 4 || p->index_bytes == 8, "index_bytes %d", p->index_bytes);
  MX_REQUIRE(p->B >= 0 && p->Nq >= 0 && p->Nk >= 0, "negative size");
  MX_REQUIRE(p->Nq <= MX_ATTENTION_MAX_ROWS && p->Nk <= MX_ATTENTION_MAX_ROWS &&
                 p->B <= MX_ATTENTION_MAX_ROWS,
             "more than %d rows or lists", MX_ATTENTION_MAX_ROWS);
  MX_REQUIRE(p->H > 0 && p->Hkv > 0 && p->H % p->Hkv == 0,
             "%d query heads are no multiple of %d key-value heads", p->H, p->Hkv);
  MX_REQUIRE(static_cast<int64_t>(p->H) * p->D <= (1ll << 23), "rows of %d heads of %d are too wide", p->H, p->D);
  MX_REQUIRE(p->D > 0 && p->D <= MX_ATTENTION_MAX_D && p->D % 8 == 0,
             "head width %d is no multiple of 8 up to %d", p->D, MX_ATTENTION_MAX_D);
  MX_REQUIRE(std::isfinite(p->scale) && p->scale > 0.0f, "scale must be positive and finite");
  // Without lists too, rows lie before or after the one entry, which the kernels read.
  MX_REQUIRE((p->q_offsets != nullptr && p->k_offsets != nullptr) || (p->B == 0 && p->Nq == 0 && p->Nk == 0),
             "offsets are null");
  return MX_OK;
}

// Tiles by rank: lists few enough for a lane each, long enough that a tile's
// length tells in the launch's, and more tiles than the chip holds at once (8
// lists of 2048, 8 heads of 64, in us: forward 70 -> 55, backward 194 -> 158; 16
// lists of 512: 24.9 either way, and 0.4 more where all start at once).
int32_t ranked_tiles(const mx_attention_problem* p) {
  return p->B > 0 && p->B + 2 <= 64 && (p->Nq + p->Nk) / p->B >= 1024 &&
         ceil_div(p->Nq, 128) * p->H > 2 * num_cus();
}

// Tiles in an order worked out by a launch of its own (about 6 us), where
// find_ranked does not serve.  In us, without and with it: ragged lists gain, lists
// of one length pay for the launch.  8 heads of 64, lists of 1 to 1000: 62 with 2
// key-value heads backward 208 -> 184, forward 55.3 -> 53.9; 32 of them backward
// 103 -> 92; 60 of 1 to 500: 71 -> 65, forward 27 -> 30; 128 of 1 to 2000: forward
// 306 -> 291; 1000 of 100: forward 189 -> 130, backward 513 -> 348; 100 of 512:
// forward 63 -> 66, backward 213 -> 216; 32 of 512, heads of 96: 122 -> 128.
bool planned_tiles(const mx_attention_problem* p, bool backward) {
  return p->B > 0 && !ranked_tiles(p) && ceil_div(p->Nq, 128) * p->H > (backward ? 2 : 16) * num_cus();
}

// Turns of the queries' and of the keys' tiles.
int64_t q_turns(const mx_attention_problem* p) { return tile_turns(p->Nq, p->B, 128 >> heads_packed(p)); }
int64_t k_turns(const mx_attention_problem* p) { return tile_turns(p->Nk, p->B, 128); }

// Each query's lse and delta, up to where turns may begin.
size_t stats_bytes(const mx_attention_problem* p) {
  return (static_cast<size_t>(p->Nq) * p->H * 2 * sizeof(float) + alignof(Turn) - 1) / alignof(Turn) * alignof(Turn);
}

// The backward's workspace: stats, turns, the shares' sums.
size_t sums_at(const mx_attention_problem* p) {
  return stats_bytes(p) + (planned_tiles(p, true) ? static_cast<size_t>(q_turns(p) + k_turns(p)) * sizeof(Turn) : 0);
}

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need > 0 && (workspace == nullptr || bytes < need))
    return mx::set_error(MX_EWORKSPACE, "workspace of %zu bytes, %zu needed", bytes, need);
  MX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % alignof(Turn) == 0, "workspace must start at a multiple of %zu bytes",
             alignof(Turn));
  return MX_OK;
}

// Writes the orders: of the queries' tiles to `turns`, and of the keys' tiles
// after them if `keys`.
int plan(const mx_attention_problem* p, Turn* turns, bool keys, hipStream_t stream) {
  PlanArgs a{};
  a.q_offsets = p->q_offsets, a.k_offsets = p->k_offsets;
  a.B = static_cast<int32_t>(p->B), a.Nq = static_cast<int32_t>(p->Nq), a.Nk = static_cast<int32_t>(p->Nk);
  a.causal = p->causal;
  a.n[0] = static_cast<int32_t>(q_turns(p));
  a.n[1] = static_cast<int32_t>(k_turns(p));
  a.shift[0] = kRowShift - heads_packed(p), a.shift[1] = kRowShift;
  a.turns[0] = turns;
  a.turns[1] = turns + a.n[0];
  const dim3 grid(keys ? 2 : 1);
  if (p->index_bytes == 8) plan_kernel<int64_t><<<grid, kPlanThreads, 0, stream>>>(a);
  else plan_kernel<int32_t><<<grid, kPlanThreads, 0, stream>>>(a);
  MX_LAUNCH_CHECK();
  return MX_OK;
}

}  // namespace
}  // namespace attn
}  // namespace mx

extern "C" size_t mx_jagged_attention_forward_workspace_bytes(const mx_attention_problem* p) {
  using namespace mx::attn;
  if (check_problem(p) != MX_OK || p->Nq == 0 || !planned_tiles(p, false)) return 0;
  return static_cast<size_t>(q_turns(p)) * sizeof(Turn);
}

extern "C" int mx_jagged_attention_forward(const mx_attention_problem* p, const mx_attention_tensor* q,
                                           const mx_attention_tensor* k, const mx_attention_tensor* v,
                                           void* out, float* lse, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_problem(p)) return rc;
  if (int rc = check_operand("q", q, p->D, p->Nq)) return rc;
  if (int rc = check_operand("k", k, p->D, p->Nk)) return rc;
  if (int rc = check_operand("v", v, p->D, p->Nk)) return rc;
  if (p->Nq == 0) return MX_OK;
  MX_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0, "out must be 16-byte aligned");
  const size_t need = mx_jagged_attention_forward_workspace_bytes(p);
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  FwdArgs a{};
  a.q = static_cast<const char*>(q->data);
  a.k = static_cast<const char*>(k->data);
  a.v = static_cast<const char*>(v->data);
  a.q_row = row_bytes(q), a.q_head = q->head_stride * 2;
  a.k_row = row_bytes(k), a.k_head = k->head_stride * 2;
  a.v_row = row_bytes(v), a.v_head = v->head_stride * 2;
  a.q_offsets = p->q_offsets, a.k_offsets = p->k_offsets;
  a.B = static_cast<int32_t>(p->B), a.Nq = static_cast<int32_t>(p->Nq), a.Nk = static_cast<int32_t>(p->Nk);
  a.H = p->H, a.G = p->H / p->Hkv, a.D = p->D;
  a.causal = p->causal, a.scale = p->scale;
  a.pack = heads_packed(p);
  a.ranked = ranked_tiles(p);
  a.out = out, a.lse = lse;
  const hipStream_t s = mx::as_stream(stream);
  if (need > 0) {
    Turn* turns = static_cast<Turn*>(workspace);
    if (int rc = plan(p, turns, false, s)) return rc;
    a.turns = turns;
    a.n_turns = static_cast<int32_t>(q_turns(p));
  }
  return p->dtype == MX_DTYPE_BF16 ? MX_ATTN_DISPATCH(launch_fwd, __bf16, a, p->index_bytes, s)
                                   : MX_ATTN_DISPATCH(launch_fwd, _Float16, a, p->index_bytes, s);
}

extern "C" size_t mx_jagged_attention_backward_workspace_bytes(const mx_attention_problem* p) {
  using namespace mx::attn;
  if (check_problem(p) != MX_OK) return 0;
  size_t n = sums_at(p);
  const int64_t shares = query_shares(p);
  if (shares > 1) n += static_cast<size_t>(shares) * 2 * p->Nk * p->Hkv * p->D * sizeof(float);
  return n;
}

extern "C" int mx_jagged_attention_backward(const mx_attention_problem* p, const mx_attention_tensor* q,
                                            const mx_attention_tensor* k, const mx_attention_tensor* v,
                                            const mx_attention_tensor* out,
                                            const mx_attention_tensor* grad_out, const float* lse,
                                            void* dq, void* dk, void* dv, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_problem(p)) return rc;
  if (int rc = check_operand("q", q, p->D, p->Nq)) return rc;
  if (int rc = check_operand("k", k, p->D, p->Nk)) return rc;
  if (int rc = check_operand("v", v, p->D, p->Nk)) return rc;
  if (int rc = check_operand("out", out, p->D, p->Nq)) return rc;
  if (int rc = check_operand("grad_out", grad_out, p->D, p->Nq)) return rc;
  MX_REQUIRE(p->Nq == 0 || (dq != nullptr && lse != nullptr), "dq or lse is null");
  MX_REQUIRE((dk == nullptr) == (dv == nullptr), "dk and dv: both or neither");
  for (const void* x : {dq, dk, dv})
    MX_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "gradients must be 16-byte aligned");
  if (int rc = check_workspace(workspace, workspace_bytes, mx_jagged_attention_backward_workspace_bytes(p)))
    return rc;
  BwdArgs a{};
  a.q = static_cast<const char*>(q->data);
  a.k = static_cast<const char*>(k->data);
  a.v = static_cast<const char*>(v->data);
  a.out = static_cast<const char*>(out->data);
  a.grad = static_cast<const char*>(grad_out->data);
  a.q_row = row_bytes(q), a.q_head = q->head_stride * 2;
  a.k_row = row_bytes(k), a.k_head = k->head_stride * 2;
  a.v_row = row_bytes(v), a.v_head = v->head_stride * 2;
  a.o_row = row_bytes(out), a.o_head = out->head_stride * 2;
  a.g_row = row_bytes(grad_out), a.g_head = grad_out->head_stride * 2;
  a.q_offsets = p->q_offsets, a.k_offsets = p->k_offsets;
  a.B = static_cast<int32_t>(p->B), a.Nq = static_cast<int32_t>(p->Nq), a.Nk = static_cast<int32_t>(p->Nk);
  a.H = p->H, a.Hkv = p->Hkv, a.G = p->H / p->Hkv, a.D = p->D;
  a.causal = p->causal, a.scale = p->scale;
  a.pack = heads_packed(p);
  a.ranked = ranked_tiles(p);
  a.lse = lse;
  a.lse2 = static_cast<float*>(workspace);
  a.delta = a.lse2 + p->Nq * p->H;
  a.dq = dq, a.dk = dk, a.dv = dv;
  const hipStream_t s = mx::as_stream(stream);
  a.shares = query_shares(p);
  a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums_at(p));
  if (planned_tiles(p, true)) {
    Turn* turns = reinterpret_cast<Turn*>(static_cast<char*>(workspace) + stats_bytes(p));
    if (int rc = plan(p, turns, dk != nullptr, s)) return rc;
    a.n_q_turns = static_cast<int32_t>(q_turns(p));
    a.n_k_turns = static_cast<int32_t>(k_turns(p));
    a.q_turns = turns;
    a.k_turns = turns + a.n_q_turns;
  }
  return p->dtype == MX_DTYPE_BF16 ? MX_ATTN_DISPATCH(launch_bwd, __bf16, a, p->index_bytes, s)
                                   : MX_ATTN_DISPATCH(launch_bwd, _Float16, a, p->index_bytes, s);
}
