// Attention of one new token per sequence over a paged cache of 4-bit rows.
//
// A row is D / 2 bytes of codes c (0..15, the even element in the low half), then
// scale s and bias b in fp16.  With e = c - 8 and f = b + 8 s a value is s e + f,
// so that over the tokens j of a sequence
//   score_j = scale (s_j (q . e_j) + f_j sum(q)),
//   out = sum_j p_j s_j e_j + sum_j p_j f_j,   p = softmax(score):
// the matrix products run on the small integers e, scale and bias enter once per
// token.
#include <type_traits>

#include "paged_common.h"
#include "row_codec.h"

namespace mx {
namespace attn {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// e = c - 8 in fp16, two at a time and exact: with the exponent of 1024 (ulp 1) set
// above it, a code in bits 0..3 of a half reads 1024 + c, one in bits 4..7 1024 + 16 c.
// The compiler knows none of the constants, or it would take two instructions with
// a literal each.  (Products on the codes as they stand, their offset taken off by
// another product, save one instruction of two but leave the offset in the sums: on
// 1024 + c, scores were off by 5e-4 and more for queries of mean 1.  On c as a
// subnormal number, of which the matrix unit keeps fewer bits, small outputs were off
// by 2^-16 of the values.)
struct Codes {
  uint32_t low, high, base;
  f16x2 sixteenth;
  __device__ __forceinline__ Codes() {
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(low));
    asm("s_mov_b32 %0, 0x00f000f0" : "=s"(high));
    asm("v_mov_b32 %0, 0x64006400" : "=v"(base));
    uint32_t x;
    asm("v_mov_b32 %0, 0x2c002c00" : "=v"(x));
    sixteenth = __builtin_bit_cast(f16x2, x);
  }
  __device__ __forceinline__ int two(uint32_t w) const {
    const f16x2 off = {-1032, -1032};
    return __builtin_bit_cast(int, __builtin_bit_cast(f16x2, (w & low) | base) + off);
  }
  __device__ __forceinline__ int two16(uint32_t w) const {
    const f16x2 off = {-72, -72};
    return __builtin_bit_cast(int, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & high) | base), sixteenth, off));
  }
};

// N values (2, 4, 8) of a row's codes, in a word's low bits.
template <int EV>
__device__ __forceinline__ uint32_t load_codes(const char* p) {
  if constexpr (EV == 8) return *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (EV == 4) return *reinterpret_cast<const uint16_t*>(p);
  else return *reinterpret_cast<const uint8_t*>(p);
}

// KS words from a multiple of 4 bytes.
template <int KS>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[KS]) {
  if constexpr (KS == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    typedef uint32_t V __attribute__((ext_vector_type(KS), aligned(4)));
    const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int s = 0; s < KS; ++s) w[s] = v[s];
  }
}

// A wave's 32 keys as they lie in memory: codes of two keys (a quarter of the row
// each) and of eight values (EV columns each), and a row's scale and bias.
template <int KS>
struct Tile4 {
  uint32_t k[2][KS], v[8], tail, seen;
};

// A power of two that brings a head's queries to where fp16 holds them with all their
// bits, and the matrix unit too (of subnormal numbers it keeps fewer).  From 1 to 2^15
// for the largest nothing is needed: what is rounded or cut then, below 2^-14, is off by
// 2^-25 of the largest at most, less than fp32 sums keep beside its product.
__device__ __forceinline__ int query_shift(float largest) {
  if (!(largest > 0.0f) || (largest >= 1.0f && largest < 32768.0f)) return 0;
  const int e = static_cast<int>(__float_as_uint(largest) >> 23) - 127;  // subnormals: -127
  return 14 - e;
}

// One block: up to 16 query heads of one key-value head, and a share of its
// tiles (or one sequence), as attention over a 16-bit cache; its waves take 32
// of a tile's keys each.  Codes go straight into registers and become fp16
// integers e there (r = lane % 16, g = lane / 16): for the scores the lane has key
// r's g-th quarter of the row, for the second product DP / 16 columns of 8 keys,
// which come out as one operand each of DP / 16 products.
//
// Queries are exact in fp16, by a power of two per head where they are large or small
// (query_shift).  p_j s_j is rounded to fp16 (2^-11), times a power of two that
// keeps the largest s seen below 128 (p stays below 256): those of an s 2^21 times
// smaller than the largest lose bits.  For fp16 outputs what the rounding leaves is a
// second operand (rounded once, they would be half as far off again as their own
// rounding makes them).
//
// Bound: reading the cache (256 sequences of 8192, 16 heads of 128 over 4: 240 us, 4.75
// TB/s, in bf16 230; the 16-bit cache 742), the issue of instructions more than half of
// the time (in fp16 281 vector and 24 matrix ones for 32 keys, in bf16 16 matrix ones; 64
// vector ones are for e instead of codes, which cost 3 to 4 percent).  64 sequences of 64 to
// 4096, 32 heads over 8: 46 us, 3.1 TB/s, of which 5 the join and
// much of the rest beginnings and ends of sequences, 4 us each.  P16 (pages of a
// multiple of 16 tokens): the wave finds addresses, else lanes do and pass them on.
// Loads past the caches are slower here (by a fifth): rows of 68 bytes share lines.
// Three blocks a CU up to D 64 (280 us for 256 of 8192, 8 heads; two took 315 and more);
// at 128 the registers would not hold it (spilled, by a quarter slower).
template <typename T, int DP, int WAVES, bool P16>
__global__ void __launch_bounds__(WAVES * 64, WAVES == kStepWaves ? (DP <= 64 ? 3 : 2) : WAVES / 4)
    step4_kernel(const StepArgs a) {
  using E = Elem<T>;
  constexpr bool kSplit = E::kNarrow;
  constexpr int kTile = WAVES * kStepKeys;
  constexpr int KS = DP / 32;  // products along D of a score; words of codes per lane
  constexpr int EV = DP / 16;  // columns of V per lane
  __shared__ float sh_o[WAVES][16][DP + 1];
  __shared__ float sh_m[WAVES][16], sh_l[WAVES][16];
  __shared__ f32x2 sh_tail[WAVES][2][kStepKeys];  // (s, f) of a tile's keys and values

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
  const int words = a.D / 8, tail = a.D / 2;
  const Codes codes;
  const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
  // Strides inside a page, and of a page, are below 2^31 bytes (checked by the host).
  const int32_t pages = static_cast<int32_t>(a.c.pages < 0x7fffffff ? a.c.pages : 0x7fffffff);
  const uint32_t k_page = static_cast<uint32_t>(a.c.k_page), v_page = static_cast<uint32_t>(a.c.v_page);
  const uint32_t k_slot = static_cast<uint32_t>(a.c.k_slot), v_slot = static_cast<uint32_t>(a.c.v_slot);
  // The lane's place in a row of codes: words word0.. of a key, the byte of its
  // first column of a value (past the row's end: the first, of a column unused).
  const int word0 = KS * g < words - KS ? KS * g : words - KS;
  const int column = EV * r < a.D ? EV * r / 2 : 0;
  // And among 16 rows of a page.
  const uint32_t k_at = r * k_slot + word0 * 4, tail_at = r * (g < 2 ? k_slot : v_slot) + tail;
  uint32_t v_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v_at[i] = (4 * g + i) * v_slot + column;

  // The share: tiles [at, stop) counted from sequence b's first one.
  const bool shared = WAVES == kStepWaves && a.workers > 0;
  Cursor cursor;
  int32_t b = worker, len;
  int64_t at = 0, stop = 0;
  if (!shared) {
    len = __builtin_amdgcn_readfirstlane(tokens_of(a, b));
    stop = tiles_of<WAVES>(len);  // 0 for an empty one: its one pass writes the zeros
  } else {
    if (!find_share(a, worker, &cursor, &at, &stop)) return;
    b = cursor.b, len = cursor.length();
  }

  while (true) {
    const int32_t n = tiles_of<WAVES>(len);
    const int32_t t0 = static_cast<int32_t>(at > 0 ? at : 0), t1 = static_cast<int32_t>(stop < n ? stop : n);
    const int32_t end = t1 * kTile < len ? t1 * kTile : len;

    i32x4 qw[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int word = word0 + s;
      qw[s] = i32x4{};
      if (r < heads && word >= KS * g)
        qw[s] = *reinterpret_cast<const i32x4*>(a.q + b * a.q_row + (head0 + r) * a.q_head + word * 16);
    }
    const int32_t* row = a.c.table + b * a.c.table_row;
    // Where the pages of 32 keys from k0 on are (P16: of 16 keys and of the next 16).
    struct Pages {
      int32_t page[2], slot[2];
    };
    auto find = [&](int32_t k0) {
      Pages x;
#pragma unroll
      for (int u = 0; u < (P16 ? 2 : 1); ++u) {
        const uint32_t key = P16 ? k0 + 16 * u : k0 + (lane & 31), size = a.c.page_size;
        const uint32_t e = a.c.page_shift >= 0 ? key >> a.c.page_shift : key / size;
        x.slot[u] = static_cast<int32_t>(key - e * size);
        x.page[u] = -1;
        if (key < static_cast<uint32_t>(end)) {
          if constexpr (P16) x.page[u] = load_scalar(row + e);
          else x.page[u] = row[e];
        }
      }
      return x;
    };
    // Asks for the rows of 32 keys.  Those of no token are read from wherever is
    // safe: what they hold never shows.
    auto load = [&](int32_t k0, const Pages& at, Tile4<KS>* x) {
      if constexpr (P16) {
        // 16 keys from a multiple of 16 are in one page: addresses are the wave's.
        const char *ka[2], *va[2];
        x->seen = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool there = at.page[u] >= 0 && at.page[u] < pages;
          const uint32_t page = there ? at.page[u] : 0, slot = there ? at.slot[u] : 0;
          const int left = end - (k0 + 16 * u);
          x->seen |= there ? (left >= 16 ? 0xffffu : (1u << left) - 1u) << (16 * u) : 0u;
          ka[u] = kb + static_cast<uint64_t>(page) * k_page + slot * k_slot;
          va[u] = vb + static_cast<uint64_t>(page) * v_page + slot * v_slot;
        }
        const char* t = g == 0 ? ka[0] : g == 1 ? ka[1] : g == 2 ? va[0] : va[1];
        x->tail = *reinterpret_cast<const uint32_t*>(t + tail_at);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          load_words<KS>(ka[u] + k_at, x->k[u]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x->v[4 * u + i] = load_codes<EV>(va[u] + v_at[i]);
        }
      } else {
        const bool there = at.page[0] >= 0 && at.page[0] < pages;
        x->seen = static_cast<uint32_t>(__ballot(there));
        const uint32_t page = there ? at.page[0] : 0, slot = there ? at.slot[0] : 0;
        const int64_t koff = static_cast<uint64_t>(page) * k_page + slot * k_slot;
        const int64_t voff = static_cast<uint64_t>(page) * v_page + slot * v_slot;
        x->tail = *reinterpret_cast<const uint32_t*>((lane < 32 ? kb + koff : vb + voff) + tail);
#pragma unroll
        for (int u = 0; u < 2; ++u) load_words<KS>(kb + shfl64(koff, 16 * u + r) + word0 * 4, x->k[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x->v[i] = load_codes<EV>(vb + shfl64(voff, 16 * (i / 4) + 4 * g + i % 4) + column);
      }
    };
    // A tile's rows are asked for one tile ahead, their pages two.
    int32_t k0 = t0 * kTile + wave * kStepKeys;
    Tile4<KS> x0, x1;
    Pages at_page = find(k0);
    if (k0 < end) load(k0, at_page, &x0);
    at_page = find(k0 + kTile);

    // Queries in the codes' order.  A row's end may cut its quarters short: they
    // begin early enough then, and what another quarter has too meets zeros.
    f16x8 qf[KS];
    f32x4 total{};
    float qx[KS][8], largest = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const typename E::x8 x = __builtin_bit_cast(typename E::x8, qw[s]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qx[s][i] = static_cast<float>(x[(i >> 1) + 4 * (i & 1)]);
        largest = fmaxf(largest, fabsf(qx[s][i]));
      }
    }
    largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
    largest = fmaxf(largest, other_half(largest));
    const int shift = query_shift(largest);
    const bool scaled = __any(shift != 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) qf[s][i] = static_cast<_Float16>(ldexpf(qx[s][i], shift));
      total = mfma(ones, qf[s], total);
    }
    const float qsum = ldexpf(total[0], -shift);  // of head r
    float most_s = 0.0f;  // the largest |s| that p s may meet, times 2^es
    int es = 0;
    float m = -INFINITY, sum = 0.0f, add = 0.0f;
    f32x4 o[EV];
#pragma unroll
    for (int t = 0; t < EV; ++t) o[t] = f32x4{};

    auto sum_up = [&](const Tile4<KS>& x) {
      const uint32_t seen = x.seen;
      {
        RowCodec<4, false> codec;
        codec.load(reinterpret_cast<const uint8_t*>(&x.tail));
        const bool here = (seen >> (lane & 31)) & 1;
        if (__any(here && lane >= 32 && fabsf(codec.scale) > most_s)) {
          float big = here && lane >= 32 ? fabsf(codec.scale) : 0.0f;
#pragma unroll
          for (int d = 1; d < 64; d *= 2) big = fmaxf(big, __shfl_xor(big, d, 64));
          // s < 2^(e + 1), and s 2^es < 128.  (A scale in fp16 is no subnormal here.)
          const int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
          most_s = ldexpf(1.0f, e + 1);
          const float f = ldexpf(1.0f, 6 - e - es);
#pragma unroll
          for (int t = 0; t < EV; ++t) o[t] *= f;
          es = 6 - e;
        }
        const float f = __builtin_fmaf(8.0f, codec.scale, codec.bias);
        const f32x2 tail = lane < 32 ? f32x2{codec.scale * c2, f * c2} : f32x2{ldexpf(codec.scale, es), f};
        sh_tail[wave][lane >> 5][lane & 31] = here ? tail : f32x2{};
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      f32x2 kt[8], vt[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) kt[i] = sh_tail[wave][0][16 * (i / 4) + 4 * g + i % 4];
      f32x4 s[2] = {};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t w = x.k[u][i], w8 = w >> 8;
          s[u] = mfma(__builtin_bit_cast(f16x8, i32x4{codes.two(w), codes.two16(w), codes.two(w8), codes.two16(w8)}),
                      qf[i], s[u]);
        }
      if (scaled) {
        asm volatile("" ::: "memory");  // a branch
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = ldexpf(s[i / 4][i % 4], -shift);
      }
      // Scores in base 2, less the maximum that runs along.
      const float mc = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        s[i / 4][i % 4] = __builtin_fmaf(kt[i][0], s[i / 4][i % 4], __builtin_fmaf(kt[i][1], qsum, -mc));
      if (seen != 0xffffffffu) {
        asm volatile("" ::: "memory");  // a branch: hardly any tile comes here
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (((seen >> (16 * u + 4 * g + i)) & 1) == 0) s[u][i] = -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                        fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      if (__any(top > (m == -INFINITY ? -INFINITY : 8.0f))) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, other_half(top));
        const float m2 = fmaxf(m, top + mc);
        const float f = m2 == -INFINITY ? 1.0f : exp2_hw(m - m2), less = m2 == -INFINITY ? 0.0f : mc - m2;
        sum *= f;
        add *= f;
#pragma unroll
        for (int t = 0; t < EV; ++t) o[t] *= f;
        // (At most 0, also where scores are so large that fp32 rounds the difference up.)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = s[i / 4][i % 4] + less;
          s[i / 4][i % 4] = x > 0.0f ? 0.0f : x;  // NaN stays
        }
        m = m2;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) vt[i] = sh_tail[wave][1][16 * (i / 4) + 4 * g + i % 4];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      f32x8 ps;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = exp2_hw(s[i / 4][i % 4]);
        sum += e;
        add = __builtin_fmaf(e, vt[i][1], add);
        ps[i] = e * vt[i][0];
      }
      const f16x8 p = __builtin_convertvector(ps, f16x8);
      f16x8 rest{};
      if constexpr (kSplit) {
        const f32x8 r8 = ps - __builtin_convertvector(p, f32x8);
        rest = __builtin_convertvector(r8, f16x8);
      }
      // Columns EV r + t of the eight keys, two to a word.
      constexpr int kHalves = EV == 8 ? 2 : 1, kPairs = EV == 2 ? 1 : 2;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(x.v[2 * i + 1], x.v[2 * i], h == 0 ? 0x05040100u : 0x07060302u);
#pragma unroll
        for (int t = 0; t < kPairs; ++t) {
          i32x4 c, c16;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t y = w[i] >> (8 * t);
            c[i] = codes.two(y);
            c16[i] = codes.two16(y);
          }
          f32x4 &even = o[4 * h + 2 * t], &odd = o[4 * h + 2 * t + 1];
          even = mfma(__builtin_bit_cast(f16x8, c), p, even);
          odd = mfma(__builtin_bit_cast(f16x8, c16), p, odd);
          if constexpr (kSplit) {
            even = mfma(__builtin_bit_cast(f16x8, c), rest, even);
            odd = mfma(__builtin_bit_cast(f16x8, c16), rest, odd);
          }
        }
      }
    };
    while (k0 < end) {
      if (k0 + kTile < end) load(k0 + kTile, at_page, &x1);
      at_page = find(k0 + 2 * kTile);
      sum_up(x0);
      k0 += kTile;
      if (k0 >= end) break;
      if (k0 + kTile < end) load(k0 + kTile, at_page, &x0);
      at_page = find(k0 + 2 * kTile);
      sum_up(x1);
      k0 += kTile;
    }

    // The waves' sums: lane (r, g) holds head r, columns EV (4 g + i) + t.
    sum += __shfl_xor(sum, 16, 64);
    sum += other_half(sum);
    add += __shfl_xor(add, 16, 64);
    add += other_half(add);
    if (g == 0) {
      sh_m[wave][r] = m;
      sh_l[wave][r] = sum;
    }
    const float unit = ldexpf(1.0f, -es);
#pragma unroll
    for (int t = 0; t < EV; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sh_o[wave][r][EV * (4 * g + i) + t] = __builtin_fmaf(o[t][i], unit, add);
    finish_block<T, WAVES, DP>(a, sh_o, sh_m, sh_l, worker, b, t0, t1, n, head0, heads);
    if (!shared || stop <= n + a.lead) return;  // a block per sequence never leaves its own
    // The next sequence that has tokens.
    stop -= n + a.lead;
    at = 0;
    if (!cursor.next(a)) return;
    b = cursor.b, len = cursor.length();
    __syncthreads();
  }
}

constexpr int wide_waves4(int D) { return D <= 32 ? 16 : 8; }  // by the registers

// How a call's sequences are cut.  Times in us, of back-to-back calls.
// - A block of four waves per sequence and head where no sequence has more than
//   eight tiles (64 of up to 1024, 8 heads of 64: 14, wide blocks 16, shares 18; of 128: 17.5, 21, 22),
//   or blocks are many and even out by themselves (1024 of up to 2048, 2 x 128: 90, in shares 100; 2048 of up
//   to 1000, 4 x 64: 74, in shares 132).  For more than 512 sequences whatever the table's
//   length: 8 percent where they are even (1024 of 8192, 8 x 64: 1,055, in shares 1,141),
//   nothing where they are not (of up to 8192 by their logarithm: 213 and 205), and one very
//   long one among them is waited for (600 of up to 500 but one of 131,072: 975, in shares 87).
// - A wide block per sequence and head where blocks are too few to fill the chip
//   and sequences short (16 of 1024, 8 x 64: 9.2, blocks of four waves 12.2, shares 14.0).
// - Else equal shares of all tiles, two blocks for every CU (three up to D 64, where
//   the registers allow it), and a second launch that joins them (256 of up to 8192
//   by their logarithm, 8 x 128: 81, a block per sequence 129; 256 of 8192 each, 8 x 64: 288, a block per
//   sequence 270: the host does not know lengths).
struct Plan {
  int32_t workers;  // 0: a block per sequence and head
  bool wide;
};

// What a sequence's beginning costs a share, in tiles: us for 64 sequences of 64 to 4096
// (32 heads of 128 over 8) with none, 1, 2, 3, 4 and 6: 50.4, 47.4, 46.0, 45.7, 46.5, 48.5; for 256 of up
// to 8192 by their logarithm (16 over 8) 100.6, 86.5, 81.0, 83.4, 88.2, 94.0.
constexpr int32_t kLead = 2;

Plan plan_step(int64_t B, int32_t heads, int32_t D, int64_t most) {
  const int64_t tiles = ceil_div(most, kTileKeys), blocks = B * heads, cus = num_cus();
  if (tiles <= 1) return {0, false};
  if (blocks > cus) {
    if (tiles <= 8 || (blocks >= 8 * cus && (tiles < 32 || B > 512))) return {0, false};
  } else if (most <= 4 * wide_waves4(D) * kStepKeys) {
    return {0, true};
  }
  const int64_t w = ceil_div(cus * (D <= 64 ? 3 : 2), heads);
  return {static_cast<int32_t>(w < B * tiles ? w : B * tiles), false};
}

template <typename T, int DP>
int launch_step(const StepArgs& a, hipStream_t s) {
  const int64_t blocks = static_cast<int64_t>(a.workers > 0 ? a.workers : a.B) * a.Hkv * a.head_blocks;
  const int64_t joins = static_cast<int64_t>(a.B) * a.H;
  MX_REQUIRE(blocks < (1ll << 22) && joins < (1ll << 22), "too many sequences: %d", a.B);  // threads in 32 bits
  auto launch = [&](auto p16) {
    constexpr bool P16 = decltype(p16)::value;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (a.wide) step4_kernel<T, DP, wide_waves4(DP), P16><<<grid, wide_waves4(DP) * 64, 0, s>>>(a);
    else step4_kernel<T, DP, kStepWaves, P16><<<grid, kStepWaves * 64, 0, s>>>(a);
  };
  if (a.c.page_size % 16 == 0) launch(std::true_type{});
  else launch(std::false_type{});
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

extern "C" size_t mx_paged_cache_attention_int4_workspace_bytes(const mx_paged_cache* cache, int64_t B, int32_t H,
                                                                int32_t Hkv, int32_t D) {
  using namespace mx::attn;
  if (cache == nullptr || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0) return 0;
  const Plan plan = plan_step(B, Hkv * head_blocks_of(H, Hkv), D, cache->table_width * cache->page_size);
  return static_cast<size_t>(plan.workers) * 2 * H * (D + 2) * sizeof(float);
}

extern "C" int mx_paged_cache_attention_int4(const mx_paged_cache* cache, int32_t dtype, const mx_attention_tensor* q,
                                             int64_t B, int32_t H, int32_t Hkv, int32_t D, const void* lengths,
                                             int32_t lengths_bytes, float scale, void* out, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_rows_cache(cache, 4)) return rc;
  MX_REQUIRE(dtype == MX_DTYPE_F16 || dtype == MX_DTYPE_BF16, "dtype %d is not fp16 or bf16", dtype);
  MX_REQUIRE(Hkv > 0 && D > 0 && D % 8 == 0 && D <= MX_ATTENTION_MAX_D, "head width %d is no multiple of 8 up to %d",
             D, MX_ATTENTION_MAX_D);
  MX_REQUIRE(B >= 0 && B < (1ll << 31), "%lld sequences", (long long)B);
  MX_REQUIRE(cache->table_width <= (1ll << 30) / cache->page_size, "more than 2^30 tokens in a row of the table");
  MX_REQUIRE(H > 0 && H % Hkv == 0, "%d query heads are no multiple of %d key-value heads", H, Hkv);
  MX_REQUIRE(std::isfinite(scale) && scale > 0.0f, "scale must be positive and finite");
  MX_REQUIRE(lengths_bytes == 4 || lengths_bytes == 8, "lengths_bytes %d", lengths_bytes);
  for (int64_t page : {cache->k_page_stride, cache->v_page_stride})
    MX_REQUIRE(page < (1ll << 31), "a page's stride is %lld bytes, 2^31 or more", (long long)page);
  for (int64_t slot : {cache->k_slot_stride, cache->v_slot_stride})
    MX_REQUIRE(slot <= ((1ll << 31) - 1) / cache->page_size, "a page's slots reach 2^31 bytes or further");
  if (B == 0) return MX_OK;
  MX_REQUIRE(q != nullptr && q->data != nullptr && out != nullptr && lengths != nullptr &&
                 (cache->table != nullptr || cache->table_width == 0),
             "null argument");
  MX_REQUIRE(reinterpret_cast<uintptr_t>(q->data) % 16 == 0 && q->row_stride % 8 == 0 && q->head_stride % 8 == 0 &&
                 q->row_stride >= 0 && q->head_stride >= 0,
             "q: rows and heads must start at multiples of 16 bytes");
  StepArgs a{};
  a.c = cache_of(cache, 1);
  a.q = static_cast<const char*>(q->data);
  a.q_row = q->row_stride * 2, a.q_head = q->head_stride * 2;
  a.lengths = lengths, a.lengths_bytes = lengths_bytes;
  a.B = static_cast<int32_t>(B), a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.D = D;
  a.head_blocks = head_blocks_of(H, Hkv);
  a.scale = scale, a.units = 1.0f;
  a.out = out;
  const Plan plan = plan_step(B, Hkv * a.head_blocks, D, cache->table_width * cache->page_size);
  a.workers = plan.workers, a.wide = plan.wide, a.lead = kLead;
  const size_t need = mx_paged_cache_attention_int4_workspace_bytes(cache, B, H, Hkv, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return mx::set_error(MX_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = mx::as_stream(stream);
  return dtype == MX_DTYPE_BF16 ? step_by_width<__bf16>(a, s) : step_by_width<_Float16>(a, s);
}
