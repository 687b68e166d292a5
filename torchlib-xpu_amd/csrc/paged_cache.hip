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
// heads of both tensors in 16-byte chunks.
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
  int32_t H, Hkv, G, D;
  int32_t head_blocks;     // of 16 query heads of a key-value head
  int32_t splits;
  int64_t chunk;           // keys of a split
  float scale;
  void* out;               // [B, H, D]
  float* part;             // [B, H, splits, D + 2]: sums, then maximum and sum of weights
};

constexpr int kStepWaves = 4;
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

// One block: a sequence, up to 16 query heads of one key-value head, one split
// of its keys; its waves take tiles of 32 keys in turn.  Every key and value is
// read once, straight into registers in the matrix operands' layouts (r = lane
// % 16, g = lane / 16): K K-major (16 keys x 32 columns per 16x16x32 product,
// a head per result column), V with 8 keys and DP / 16 columns per lane,
// transposed in registers.
template <typename T, int DP>
__global__ void __launch_bounds__(kStepWaves * 64) step_kernel(const StepArgs a) {
  using E = Elem<T>;
  using X8 = typename E::x8;
  constexpr int KS = DP / 32;  // products along D of a score
  constexpr int EV = DP / 16;  // columns of V per lane
  using VP = typename Piece<EV>::type;
  __shared__ float sh_o[kStepWaves][16][DP + 1];
  __shared__ float sh_m[kStepWaves][16], sh_l[kStepWaves][16];

  const int hb = blockIdx.x % a.head_blocks;
  const int64_t y = blockIdx.x / a.head_blocks;
  const int kvh = static_cast<int>(y % a.Hkv);
  const int64_t z = y / a.Hkv;
  const int split = static_cast<int>(z % a.splits);
  const int64_t b = z / a.splits;
  int64_t len = uniform64(ld_index(a.lengths, a.lengths_bytes, b));
  const int64_t most = a.c.width * a.c.page_size;
  len = len < most ? len : most;
  const int64_t begin = split * a.chunk;
  if (begin >= len && split > 0) return;
  const int64_t end = begin + a.chunk < len ? begin + a.chunk : len;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int head0 = kvh * a.G + hb * 16;
  const int heads = a.G - hb * 16 < 16 ? a.G - hb * 16 : 16;

  X8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int col = 32 * s + 8 * g;
    i32x4 w{};
    if (r < heads && col < a.D)
      w = *reinterpret_cast<const i32x4*>(a.q + b * a.q_row + (head0 + r) * a.q_head + col * 2);
    qf[s] = __builtin_bit_cast(X8, w);
  }

  const float c2 = a.scale * kLog2e;
  float m = -INFINITY, sum = 0.0f;
  f32x4 o[EV];
#pragma unroll
  for (int t = 0; t < EV; ++t) o[t] = f32x4{};
  const int32_t* row = a.c.table + b * a.c.table_row;
  const char* kb = a.c.k + kvh * a.c.k_head;
  const char* vb = a.c.v + kvh * a.c.v_head;

  for (int64_t k0 = begin + wave * kStepKeys; k0 < end; k0 += kStepWaves * kStepKeys) {
    // Lane i finds the place of key k0 + i % 32.
    const int64_t key = k0 + (lane & 31);
    int slot = 0;
    int64_t page = -1;
    if (key < end) page = row[page_of(a.c, key, &slot)];
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
        if (col < a.D) kw[u][s] = *reinterpret_cast<const i32x4*>(p + col * 2);
      }
    }
    VP vw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = 16 * (i / 4) + 4 * g + i % 4;
      const char* p = vb + shfl64(voff, n);
      vw[i] = VP{};
      if (EV * r < a.D && ((seen >> n) & 1)) vw[i] = *reinterpret_cast<const VP*>(p + EV * r * 2);
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
  for (int u = tid; u < heads * a.D; u += kStepWaves * 64) {
    const int n = u / a.D, d = u - n * a.D;
    float mm = sh_m[0][n];
#pragma unroll
    for (int w = 1; w < kStepWaves; ++w) mm = fmaxf(mm, sh_m[w][n]);
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) {
      const float f = mm == -INFINITY ? 0.0f : exp2_hw((sh_m[w][n] - mm) * c2);
      acc += f * sh_o[w][n][d];
      l += f * sh_l[w][n];
    }
    const int64_t at = b * a.H + head0 + n;
    if (a.splits == 1) {
      static_cast<T*>(a.out)[at * a.D + d] = static_cast<T>(l == 0.0f ? 0.0f : acc / l);
    } else {
      float* to = a.part + (at * a.splits + split) * (a.D + 2);
      to[d] = acc;
      if (d == 0) {
        to[a.D] = mm;
        to[a.D + 1] = l;
      }
    }
  }
}

// Joins the splits of a sequence and head, in their order: one wave each.
template <typename T>
__global__ void __launch_bounds__(64) join_kernel(const StepArgs a) {
  const int64_t at = blockIdx.x;
  const int64_t b = at / a.H;
  int64_t len = ld_index(a.lengths, a.lengths_bytes, b);
  const int64_t most = a.c.width * a.c.page_size;
  len = len < most ? len : most;
  int n = len > 0 ? static_cast<int>((len + a.chunk - 1) / a.chunk) : 1;
  n = n < a.splits ? n : a.splits;
  const float* part = a.part + at * a.splits * (a.D + 2);
  const float c2 = a.scale * kLog2e;
  float mm = -INFINITY;
  for (int s = 0; s < n; ++s) mm = fmaxf(mm, part[s * (a.D + 2) + a.D]);
  for (int d = threadIdx.x; d < a.D; d += 64) {
    float acc = 0.0f, l = 0.0f;
    for (int s = 0; s < n; ++s) {
      const float* p = part + s * (a.D + 2);
      const float f = mm == -INFINITY ? 0.0f : exp2_hw((p[a.D] - mm) * c2);
      acc += f * p[d];
      l += f * p[a.D + 1];
    }
    static_cast<T*>(a.out)[at * a.D + d] = static_cast<T>(l == 0.0f ? 0.0f : acc / l);
  }
}

// Splits of the keys: enough blocks to fill the chip, of at least 256 keys.
void plan_splits(int64_t B, int32_t Hkv, int32_t head_blocks, int64_t most, int32_t* splits, int64_t* chunk) {
  const int64_t blocks = B * Hkv * head_blocks;
  const int64_t want = blocks > 0 ? ceil_div(static_cast<int64_t>(num_cus()) * 4, blocks) : 1;
  int64_t c = ceil_div(ceil_div(most, want > 0 ? want : 1), 128) * 128;
  if (c < 256) c = 256;
  *chunk = c;
  *splits = static_cast<int32_t>(most > 0 ? ceil_div(most, c) : 1);
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
int launch_step(const StepArgs& a, int64_t B, hipStream_t s) {
  const int64_t blocks = B * a.splits * a.Hkv * a.head_blocks;
  MX_REQUIRE(blocks < (1ll << 31) && B * a.H < (1ll << 31), "too many sequences: %lld", (long long)B);
  step_kernel<T, DP><<<dim3(static_cast<unsigned>(blocks)), kStepWaves * 64, 0, s>>>(a);
  if (a.splits > 1) join_kernel<T><<<dim3(static_cast<unsigned>(B * a.H)), 64, 0, s>>>(a);
  MX_LAUNCH_CHECK();
  return MX_OK;
}

template <typename T>
int step_by_width(const StepArgs& a, int64_t B, hipStream_t s) {
  if (a.D <= 32) return launch_step<T, 32>(a, B, s);
  if (a.D <= 64) return launch_step<T, 64>(a, B, s);
  return launch_step<T, 128>(a, B, s);
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
  MX_REQUIRE(blocks < (1ll << 31), "too many rows: %lld", (long long)N);
  append_kernel<<<dim3(static_cast<unsigned>(blocks)), kAppendWaves * 64, 0, mx::as_stream(stream)>>>(a);
  MX_LAUNCH_CHECK();
  return MX_OK;
}

extern "C" size_t mx_paged_cache_attention_workspace_bytes(const mx_paged_cache* cache, int64_t B,
                                                           int32_t H, int32_t Hkv, int32_t D) {
  using namespace mx::attn;
  if (cache == nullptr || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0) return 0;
  int32_t splits = 1;
  int64_t chunk = 0;
  plan_splits(B, Hkv, head_blocks_of(H, Hkv), cache->table_width * cache->page_size, &splits, &chunk);
  return splits == 1 ? 0 : static_cast<size_t>(B) * H * splits * (D + 2) * sizeof(float);
}

extern "C" int mx_paged_cache_attention(const mx_paged_cache* cache, int32_t dtype,
                                        const mx_attention_tensor* q, int64_t B, int32_t H,
                                        int32_t Hkv, int32_t D, const void* lengths,
                                        int32_t lengths_bytes, float scale, void* out,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_cache(cache, dtype, Hkv, D)) return rc;
  MX_REQUIRE(B >= 0, "negative size");
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
  a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.D = D;
  a.head_blocks = head_blocks_of(H, Hkv);
  a.scale = scale;
  a.out = out;
  plan_splits(B, Hkv, a.head_blocks, cache->table_width * cache->page_size, &a.splits, &a.chunk);
  const size_t need = mx_paged_cache_attention_workspace_bytes(cache, B, H, Hkv, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return mx::set_error(MX_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = mx::as_stream(stream);
  return dtype == MX_DTYPE_BF16 ? step_by_width<__bf16>(a, B, s) : step_by_width<_Float16>(a, B, s);
}
