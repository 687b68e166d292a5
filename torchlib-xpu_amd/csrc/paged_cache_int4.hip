// Attention of one new token per sequence over a paged cache of 4-bit rows.
//
// A row is D / 2 bytes of codes c (0..15, the even element in the low half), then
// scale s and bias b in fp16.  With e = c - 8 and f = b + 8 s a value is s e + f,
// so that over the tokens j of a sequence
//   score_j = scale (s_j (q . e_j) + f_j sum(q)),
//   out = sum_j p_j s_j e_j + sum_j p_j f_j,   p = softmax(score):
// the matrix products run on the codes themselves, scale and bias enter once per
// token.
#include <type_traits>

#include "paged_common.h"
#include "row_codec.h"

namespace mx {
namespace attn {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 128 + c as bf16 (exponent 7, seven bits of mantissa): a code in the low bits of
// each half of a word, in one instruction for two (the compiler knows neither
// constant, or it would take two instructions with a literal each).
struct Codes {
  uint32_t mask, one28;
  __device__ __forceinline__ Codes() {
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(mask));
    asm("v_mov_b32 %0, 0x43004300" : "=v"(one28));
  }
  __device__ __forceinline__ int two(uint32_t w) const { return static_cast<int>((w & mask) | one28); }
};
constexpr float kOffset = 136.0f;  // 128 + c - 136 = c - 8

__device__ __forceinline__ bf16x8 splat(float v) {
  const __bf16 x = static_cast<__bf16>(v);
  return bf16x8{x, x, x, x, x, x, x, x};
}

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

// One block: up to 16 query heads of one key-value head, and a share of its
// tiles (or one sequence), as attention over a 16-bit cache; its waves take 32
// of a tile's keys each.  Codes go straight into registers and become bf16
// integers there (r = lane % 16, g = lane / 16): for the scores the lane has key
// r's g-th quarter of the row, for the second product DP / 16 columns of 8 keys,
// which come out as one operand each of DP / 16 products.  The integers are
// 128 + c; -136 times the other operand's sum starts each product off, so that
// what is summed is c - 8 and no more than a tile's offset ever stands in a sum.
// fp16 queries, and p_j s_j, are split into two bf16 parts.
template <typename T, int DP, int WAVES, bool P16>
__global__ void __launch_bounds__(WAVES * 64, WAVES == kStepWaves ? 2 : WAVES / 4) step4_kernel(const StepArgs a) {
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
  // The lane's place in a row of codes: words word0.. of a key, the byte of its
  // first column of a value (past the row's end: the first, of a column unused).
  const int word0 = KS * g < words - KS ? KS * g : words - KS;
  const int column = EV * r < a.D ? EV * r / 2 : 0;
  // And among 16 rows of a page.
  const int64_t k_at = r * a.c.k_slot + word0 * 4, tail_at = r * (g < 2 ? a.c.k_slot : a.c.v_slot) + tail;
  int64_t v_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v_at[i] = (4 * g + i) * a.c.v_slot + column;

  // The share: tiles [at, stop) counted from sequence b's first one.
  const bool shared = WAVES == kStepWaves && a.workers > 0;
  int32_t b = worker, len;
  int64_t at = 0, stop = 0;
  if (!shared) {
    len = __builtin_amdgcn_readfirstlane(tokens_of(a, b));
    stop = tiles_of<WAVES>(len);  // 0 for an empty one: its one pass writes the zeros
  } else if (!find_share(a, worker, &b, &len, &at, &stop)) {
    return;
  }

  while (true) {
    const int32_t n = tiles_of<WAVES>(len);
    const int32_t t0 = static_cast<int32_t>(at), t1 = static_cast<int32_t>(stop < n ? stop : n);
    const int32_t end = t1 * kTile < len ? t1 * kTile : len;

    // Queries in the codes' order: a word's halves hold codes 0 4, 1 5, 2 6, 3 7.
    // A row's end may cut its quarters short: they begin early enough then, and
    // what another quarter has too meets zeros.
    bf16x8 qf[KS], ql[KS];
    f32x4 total{};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int word = word0 + s;
      i32x4 w{};
      if (r < heads && word >= KS * g)
        w = *reinterpret_cast<const i32x4*>(a.q + b * a.q_row + (head0 + r) * a.q_head + word * 16);
      const typename E::x8 x = __builtin_bit_cast(typename E::x8, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const T v = x[(i >> 1) + 4 * (i & 1)];
        qf[s][i] = static_cast<__bf16>(static_cast<float>(v));
        if constexpr (kSplit) ql[s][i] = static_cast<__bf16>(static_cast<float>(v) - static_cast<float>(qf[s][i]));
      }
      total = mfma(splat(1.0f), qf[s], total);
      if constexpr (kSplit) total = mfma(splat(1.0f), ql[s], total);
    }
    const float qsum = total[0];  // of head r
    const float start = -kOffset * qsum;
    float m = -INFINITY, sum = 0.0f, add = 0.0f;
    f32x4 o[EV];
#pragma unroll
    for (int t = 0; t < EV; ++t) o[t] = f32x4{};

    const int32_t* row = a.c.table + b * a.c.table_row;
    // Asks for the rows of 32 keys from k0 on.  Those of no token are read from
    // wherever is safe: what they hold never shows.
    auto load = [&](int32_t k0, Tile4<KS>* x) {
      if constexpr (P16) {
        // 16 keys from a multiple of 16 are in one page: addresses are the wave's.
        const char *ka[2], *va[2];
        x->seen = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int32_t key = k0 + 16 * u;
          const uint32_t size = a.c.page_size;
          const uint32_t e = a.c.page_shift >= 0 ? static_cast<uint32_t>(key) >> a.c.page_shift : key / size;
          const int32_t slot = key - e * size;
          int32_t page = key < end ? load_scalar(row + e) : -1;
          const bool there = page >= 0 && page < a.c.pages;
          page = there ? page : 0;
          const int left = end - key;
          x->seen |= there ? (left >= 16 ? 0xffffu : (1u << left) - 1u) << (16 * u) : 0u;
          ka[u] = kb + page * a.c.k_page + (there ? slot : 0) * a.c.k_slot;
          va[u] = vb + page * a.c.v_page + (there ? slot : 0) * a.c.v_slot;
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
        const uint32_t key = k0 + (lane & 31), size = a.c.page_size;
        const uint32_t e = a.c.page_shift >= 0 ? key >> a.c.page_shift : key / size;
        const int64_t page = key < static_cast<uint32_t>(end) ? row[e] : -1;
        const bool there = page >= 0 && page < a.c.pages;
        x->seen = static_cast<uint32_t>(__ballot(there));
        const int32_t slot = key - e * size;
        const int64_t koff = there ? page * a.c.k_page + slot * a.c.k_slot : 0;
        const int64_t voff = there ? page * a.c.v_page + slot * a.c.v_slot : 0;
        x->tail = *reinterpret_cast<const uint32_t*>((lane < 32 ? kb + koff : vb + voff) + tail);
#pragma unroll
        for (int u = 0; u < 2; ++u) load_words<KS>(kb + shfl64(koff, 16 * u + r) + word0 * 4, x->k[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x->v[i] = load_codes<EV>(vb + shfl64(voff, 16 * (i / 4) + 4 * g + i % 4) + column);
      }
    };
    auto sum_up = [&](const Tile4<KS>& x) {
      const uint32_t seen = x.seen;
      {
        RowCodec<4, false> codec;
        codec.load(reinterpret_cast<const uint8_t*>(&x.tail));
        const float f = __builtin_fmaf(8.0f, codec.scale, codec.bias);
        sh_tail[wave][lane >> 5][lane & 31] = (seen >> (lane & 31)) & 1 ? f32x2{codec.scale, f} : f32x2{};
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      f32x2 kt[8], vt[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int nk = 16 * (i / 4) + 4 * g + i % 4;
        kt[i] = sh_tail[wave][0][nk];
        vt[i] = sh_tail[wave][1][nk];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();

      f32x4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) s[u] = f32x4{start, start, start, start};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t w = x.k[u][i];
          const bf16x8 c = __builtin_bit_cast(
              bf16x8, i32x4{codes.two(w), codes.two(w >> 4), codes.two(w >> 8), codes.two(w >> 12)});
          s[u] = mfma(c, qf[i], s[u]);
          if constexpr (kSplit) s[u] = mfma(c, ql[i], s[u]);
        }
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = __builtin_fmaf(kt[i][0], s[i / 4][i % 4], kt[i][1] * qsum);
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
      if (__any((top - m) * c2 > 8.0f)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, other_half(top));
        const float m2 = fmaxf(m, top);
        const float f = m2 == -INFINITY ? 1.0f : exp2_hw((m - m2) * c2);
        sum *= f;
        add *= f;
#pragma unroll
        for (int t = 0; t < EV; ++t) o[t] *= f;
        m = m2;
      }
      const float mc = m == -INFINITY ? 0.0f : m * c2;
      f32x8 ps;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = exp2_hw(__builtin_fmaf(s[i / 4][i % 4], c2, -mc));
        sum += e;
        add = __builtin_fmaf(e, vt[i][1], add);
        ps[i] = e * vt[i][0];
      }
      const bf16x8 p = __builtin_convertvector(ps, bf16x8);
      const bf16x8 pl = __builtin_convertvector(ps - __builtin_convertvector(p, f32x8), bf16x8);
      const bf16x8 minus = splat(-kOffset);
#pragma unroll
      for (int t = 0; t < EV; ++t) o[t] = mfma(minus, p, o[t]);
#pragma unroll
      for (int t = 0; t < EV; ++t) o[t] = mfma(minus, pl, o[t]);
      // Columns EV r + t of the eight keys, two to a word.
      constexpr int kHalves = EV == 8 ? 2 : 1, kColumns = EV == 8 ? 4 : EV;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(x.v[2 * i + 1], x.v[2 * i], h == 0 ? 0x05040100u : 0x07060302u);
#pragma unroll
        for (int t = 0; t < kColumns; ++t) {
          i32x4 c;
#pragma unroll
          for (int i = 0; i < 4; ++i) c[i] = codes.two(w[i] >> (4 * t));
          const bf16x8 y = __builtin_bit_cast(bf16x8, c);
          o[4 * h + t] = mfma(y, p, o[4 * h + t]);
          o[4 * h + t] = mfma(y, pl, o[4 * h + t]);
        }
      }
    };
    // A tile's rows are asked for one tile ahead.
    int32_t k0 = t0 * kTile + wave * kStepKeys;
    if (k0 < end) {
      Tile4<KS> x0, x1;
      load(k0, &x0);
      while (true) {
        if (k0 + kTile < end) load(k0 + kTile, &x1);
        sum_up(x0);
        k0 += kTile;
        if (k0 >= end) break;
        if (k0 + kTile < end) load(k0 + kTile, &x0);
        sum_up(x1);
        k0 += kTile;
        if (k0 >= end) break;
      }
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
#pragma unroll
    for (int t = 0; t < EV; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sh_o[wave][r][EV * (4 * g + i) + t] = o[t][i] + add;
    finish_block<T, WAVES, DP>(a, sh_o, sh_m, sh_l, worker, b, t0, t1, n, head0, heads);
    if (!shared || stop <= n) return;  // a block per sequence never leaves its own
    // The next sequence that has tokens.
    stop -= n;
    at = 0;
    if (!next_sequence(a, &b, &len)) return;
    __syncthreads();
  }
}

// How a call's sequences are cut: as for the 16-bit cache.
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

template <typename T, int DP>
int launch_step(const StepArgs& a, hipStream_t s) {
  const int64_t blocks = static_cast<int64_t>(a.workers > 0 ? a.workers : a.B) * a.Hkv * a.head_blocks;
  const int64_t joins = static_cast<int64_t>(a.B) * a.H;
  MX_REQUIRE(blocks < (1ll << 22) && joins < (1ll << 22), "too many sequences: %d", a.B);  // threads in 32 bits
  auto launch = [&](auto p16) {
    constexpr bool P16 = decltype(p16)::value;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (a.wide) step4_kernel<T, DP, wide_waves(DP), P16><<<grid, wide_waves(DP) * 64, 0, s>>>(a);
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
  a.scale = scale;
  a.out = out;
  const Plan plan = plan_step(B, Hkv * a.head_blocks, D, cache->table_width * cache->page_size);
  a.workers = plan.workers, a.wide = plan.wide;
  const size_t need = mx_paged_cache_attention_int4_workspace_bytes(cache, B, H, Hkv, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return mx::set_error(MX_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = mx::as_stream(stream);
  return dtype == MX_DTYPE_BF16 ? step_by_width<__bf16>(a, s) : step_by_width<_Float16>(a, s);
}
