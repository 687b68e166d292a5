// Packed rows by their positions: rotation of heads by position (and back), the
// same on the way into a paged cache, rows of a 4-bit cache, and the rows of
// lists out of a cache again.
//
// A row of list b at i behind the list's first has position p = starts[b] + i.
// Rotation turns pairs (x1, x2) of a head's first R values by the angle of
// their frequency at p, (c, s) = table[p][pair]:
//   y1 = x1 c - x2 s,   y2 = x2 c + x1 s;
// its gradient is the rotation by -angle.  Pairs are (i, i + R / 2), or (2 i,
// 2 i + 1) where interleaved.  Every product and sum is rounded to fp32 by
// itself (no fused multiply-add), so that the codes of a 4-bit row, which a last
// bit can decide, are those of the formulas.
//
// A row of a 4-bit cache is D / 2 bytes of codes (the even element in the low
// half), fp16 scale, fp16 bias: value = scale code + bias, as the 4-bit codec op
// writes rows; but for values that hold a NaN, whose row is NaN in scale and bias.
#include "paged_common.h"
#include "row_codec.h"
#include "token_of_row.h"

namespace mx {
namespace attn {
namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Quad;
template <>
struct Quad<__bf16> { using type = bf16x4; };
template <>
struct Quad<_Float16> { using type = f16x4; };

enum Kind { kRotate, kAppend16, kAppend4, kGather16, kGather4 };

struct RowsArgs {
  Cache c;
  const char* src[3];                       // q, k, v (rotation alone: x)
  int64_t src_row[3], src_head[3];          // bytes
  char* out[2];                             // rotated q; keys and values of a gather
  const void *offsets, *starts;
  int32_t offsets_bytes, starts_bytes;
  int64_t B, N;
  int32_t H, Hkv, D;                        // H: heads of src[0] (0: none)
  int32_t vecs;                             // heads of a row, of all tensors
  uint32_t vecs_inverse;                    // ceil(2^32 / vecs)
  int32_t tile_rows;                        // rows of a wave
  int32_t slices;                           // waves that share a tile's heads
  int64_t waves;
  const float* table;                       // [positions, pairs, 2] cos, sin
  int64_t positions;
  int32_t pairs, interleaved;               // pairs 0: no rotation
  float sign;                               // of the angles
};

// Where a row's heads go: its position (kNoList: in no list; kNoAngle: no entry of
// the table), and its slot in the caches (-1: it has none).
constexpr int32_t kNoList = -2, kNoAngle = -1;
struct Place {
  int32_t pos;
  int64_t k, v;
};

// The list of row r0 + lane, for lanes < rows: one search for the first row's,
// then the ends that follow.
__device__ __forceinline__ int64_t lists_of_rows(const RowsArgs& a, int64_t r0, int rows) {
  const int64_t b0 = list_of_row(a.offsets, a.offsets_bytes, a.B, r0);
  if (rows == 1) return b0;
  const int64_t i = b0 + 1 + lane_id();
  const int64_t end = i <= a.B ? ld_index(a.offsets, a.offsets_bytes, i) - r0 : 64;
  const uint64_t inside = __ballot(end < rows);
  if (inside == ~0ull) {  // many empty lists: each row by itself
    int64_t b = b0;
    for (int r = 1; r < rows; ++r) {
      const int64_t x = list_of_row(a.offsets, a.offsets_bytes, a.B, r0 + r);
      if (lane_id() == r) b = x;
    }
    return b;
  }
  int64_t b = b0;
  const int n = __popcll(inside);  // offsets do not decrease: the first n
  for (int j = 0; j < n; ++j)
    if (readlane_i32(static_cast<int32_t>(end), j) <= lane_id()) b = b0 + 1 + j;
  return b;
}

template <Kind KIND>
__device__ __forceinline__ Place place_of(const RowsArgs& a, int64_t b, int64_t row) {
  Place p{kNoList, -1, -1};
  if (b < 0 || b >= a.B || row >= a.N) return p;
  const int64_t start = a.starts != nullptr ? ld_index(a.starts, a.starts_bytes, b) : 0;
  const int64_t t = token_of_row(start, row, ld_index(a.offsets, a.offsets_bytes, b));
  p.pos = t >= 0 && t < a.positions ? static_cast<int32_t>(t) : kNoAngle;
  if constexpr (KIND != kRotate) {
    int slot;
    const int64_t e = t >= 0 ? page_of(a.c, t, &slot) : a.c.width;
    if (e < a.c.width && (a.pairs == 0 || p.pos >= 0)) {
      const int64_t page = a.c.table[b * a.c.table_row + e];
      if (page >= 0 && page < a.c.pages) {
        p.k = page * a.c.k_page + slot * a.c.k_slot;
        p.v = page * a.c.v_page + slot * a.c.v_slot;
      }
    }
  }
  return p;
}

// The places of a wave's rows: lane i holds row r0 + i's (ONE: all lanes r0's).
template <Kind KIND, bool ONE>
__device__ __forceinline__ Place places(const RowsArgs& a, int64_t r0, int rows) {
  if constexpr (ONE) {
    return place_of<KIND>(a, list_of_row(a.offsets, a.offsets_bytes, a.B, r0), r0);
  } else {
    const int64_t b = lists_of_rows(a, r0, rows);
    return place_of<KIND>(a, lane_id() < rows ? b : -1, r0 + lane_id());
  }
}

template <bool ONE>
__device__ __forceinline__ Place at_row(const Place& p, int row) {
  if constexpr (ONE) return p;
  return {__shfl(p.pos, row, 64), shfl64(p.k, row), shfl64(p.v, row)};
}

// Four pairs of a head, by four cosines and sines.
__device__ __forceinline__ void turn(float (&x)[8], const f32x4& lo, const f32x4& hi, bool interleaved, float sign) {
#pragma clang fp contract(off)
  const float c[4] = {lo[0], lo[2], hi[0], hi[2]}, s[4] = {lo[1] * sign, lo[3] * sign, hi[1] * sign, hi[3] * sign};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x1 = interleaved ? x[2 * e] : x[e], x2 = interleaved ? x[2 * e + 1] : x[4 + e];
    const float a = x1 * c[e], b = x2 * s[e], d = x2 * c[e], f = x1 * s[e];
    const float y1 = fp32_value(a - b), y2 = fp32_value(d + f);
    if (interleaved) x[2 * e] = y1, x[2 * e + 1] = y2;
    else x[e] = y1, x[4 + e] = y2;
  }
}

template <int GS>
__device__ __forceinline__ float group_min(float v) {
#pragma unroll
  for (int m = GS / 2; m >= 1; m >>= 1) v = fminf(v, __shfl_xor(v, m, 64));
  return v;
}
template <int GS>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int m = GS / 2; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

constexpr int kRowsWaves = 4;

// The wave's tile and slice; false if it has none.
struct WaveTile {
  int64_t r0;
  int rows, slice;
};
__device__ __forceinline__ bool wave_tile(const RowsArgs& a, WaveTile* t) {
  const int64_t w = uniform64(static_cast<int64_t>(blockIdx.x) * kRowsWaves + (threadIdx.x >> 6));
  if (w >= a.waves) return false;
  const int64_t tile = w / a.slices;
  t->slice = static_cast<int>(w - tile * a.slices);
  t->r0 = tile * a.tile_rows;
  t->rows = static_cast<int>(a.N - t->r0 < a.tile_rows ? a.N - t->r0 : a.tile_rows);
  return true;
}

// A wave takes tile_rows rows (ONE: one); GS lanes take a head, eight values
// each: four pairs, or eight values that do not turn (16 bytes at a time where they
// lie together: 256 lists of up to 512, 16 heads of 96, both ways, 69.7 -> 65.6 us in
// calls one after another).  Bound: the copy, for batches that fill the chip (4 lists
// of 4096, 20 heads of 128, one way: 39 us, 4.3 TB/s; appends of 32 lists of up to
// 2000, 32 heads of 128: 108 us, 4.8 TB/s, into 4-bit rows 112, 3.8 TB/s); few rows
// by the loads in turn before them (64 rows of 48 heads: 4.1 us).  Many short waves
// hide these loads best: waves of four or more rows that ask for the next heads
// beforehand took 74 for 65 us, 120 to 138 for 105.
template <typename T, int GS, Kind KIND, bool ONE>
__global__ void __launch_bounds__(kRowsWaves * 64) rows_kernel(const RowsArgs a) {
  using X4 = typename Quad<T>::type;
  using X8 = typename Elem<T>::x8;
  constexpr int kGroups = 64 / GS;
  WaveTile w;
  if (!wave_tile(a, &w)) return;
  const Place mine = places<KIND, ONE>(a, w.r0, w.rows);
  const int lane = lane_id(), group = lane / GS, u = lane % GS;
  const bool unit = 8 * u < a.D;
  const int total = w.rows * a.vecs;
  for (int p = w.slice; p * kGroups < total; p += a.slices) {
    const int t = p * kGroups + group;
    const bool in = t < total;
    int row = 0;
    if constexpr (!ONE) row = in ? (a.vecs == 1 ? t : static_cast<int>(__umulhi(t, a.vecs_inverse))) : 0;
    const int vec = t - row * a.vecs;
    const Place at = at_row<ONE>(mine, row);
    const int which = vec < a.H ? 0 : vec < a.H + a.Hkv ? 1 : 2;
    const int h = which == 0 ? vec : which == 1 ? vec - a.H : vec - a.H - a.Hkv;
    const int64_t to = which == 1 ? at.k : at.v;
    // What is dropped is not read either.
    const bool live = in && unit && (which == 0 || to >= 0);
    const bool turns = which < 2 && 4 * u < a.pairs;
    const bool split = turns && !a.interleaved;
    const int ea = split ? 4 * u : 8 * u, eb = split ? a.pairs + 4 * u : 8 * u + 4;
    float x[8];
    if (live) {
      const char* s = which == 0 ? a.src[0] + (w.r0 + row) * a.src_row[0] + h * a.src_head[0]
                      : which == 1 ? a.src[1] + (w.r0 + row) * a.src_row[1] + h * a.src_head[1]
                                   : a.src[2] + (w.r0 + row) * a.src_row[2] + h * a.src_head[2];
      X4 xa, xb;
      if (split) {
        xa = *reinterpret_cast<const X4*>(s + ea * 2), xb = *reinterpret_cast<const X4*>(s + eb * 2);
      } else {
        const X8 v = *reinterpret_cast<const X8*>(s + u * 16);
        xa = __builtin_shufflevector(v, v, 0, 1, 2, 3), xb = __builtin_shufflevector(v, v, 4, 5, 6, 7);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(xa[e]), x[4 + e] = static_cast<float>(xb[e]);
      if (turns) {
        if (at.pos >= 0) {
          const f32x4* cs = reinterpret_cast<const f32x4*>(a.table + (static_cast<int64_t>(at.pos) * a.pairs + 4 * u) * 2);
          turn(x, cs[0], cs[1], a.interleaved, a.sign);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = NAN;
        }
      }
      if (which == 0 && at.pos == kNoList) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
      }
    }
    if (KIND == kAppend4) {
      // All lanes of the group hold one head's values (or none do).
      float lo = INFINITY, hi = -INFINITY;
      bool nan = false;
      if (live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]), nan |= __builtin_isnan(x[e]);
      }
      lo = group_min<GS>(lo);
      hi = group_max<GS>(hi);
      // A code cannot say NaN, and the minimum and maximum pass over it: the head's whole row
      // is one, by its scale and bias.
      if ((__ballot(nan) >> (group * GS)) & ((1ull << GS) - 1)) lo = hi = NAN;
      if (live && which > 0) {
        RowCodec<4, false> codec;
        codec.set(lo, hi);
        uint32_t wa = 0, wb = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) wa |= codec.code(x[e]) << (4 * e), wb |= codec.code(x[4 + e]) << (4 * e);
        char* d = (which == 1 ? a.c.k + to + h * a.c.k_head : a.c.v + to + h * a.c.v_head);
        if (split) {
          *reinterpret_cast<uint16_t*>(d + ea / 2) = static_cast<uint16_t>(wa);
          *reinterpret_cast<uint16_t*>(d + eb / 2) = static_cast<uint16_t>(wb);
        } else {
          *reinterpret_cast<uint32_t*>(d + u * 4) = wa | (wb << 16);
        }
        if (u == 0) codec.store(reinterpret_cast<uint8_t*>(d) + a.D / 2);
      }
    }
    if (live && (KIND != kAppend4 || which == 0)) {
      char* d = which == 0 ? a.out[0] + ((w.r0 + row) * a.H + h) * a.D * 2
                : which == 1 ? a.c.k + to + h * a.c.k_head
                             : a.c.v + to + h * a.c.v_head;
      X4 ya, yb;
#pragma unroll
      for (int e = 0; e < 4; ++e) ya[e] = static_cast<T>(x[e]), yb[e] = static_cast<T>(x[4 + e]);
      if (split) {
        *reinterpret_cast<X4*>(d + ea * 2) = ya;
        *reinterpret_cast<X4*>(d + eb * 2) = yb;
      } else {
        *reinterpret_cast<X8*>(d + u * 16) = __builtin_shufflevector(ya, yb, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  }
}

// The lists' rows out of the pages, packed: row i of list b is its token i; zeros
// where there is no page.  Bound: the copy (16 lists of up to 2250, 8 heads of 128:
// 21 us from 4-bit rows, 4.4 TB/s, and 30 us from 16-bit ones, 4.8 TB/s).
template <typename T, int GS, Kind KIND, bool ONE>
__global__ void __launch_bounds__(kRowsWaves * 64) gather_kernel(const RowsArgs a) {
  using X8 = typename Elem<T>::x8;
  constexpr int kGroups = 64 / GS;
  WaveTile w;
  if (!wave_tile(a, &w)) return;
  const Place mine = places<KIND, ONE>(a, w.r0, w.rows);
  const int lane = lane_id(), group = lane / GS, u = lane % GS;
  const bool unit = 8 * u < a.D;
  const int total = w.rows * a.vecs;
  for (int p = w.slice; p * kGroups < total; p += a.slices) {
    const int t = p * kGroups + group;
    const bool in = t < total;
    int row = 0;
    if constexpr (!ONE) row = in ? static_cast<int>(__umulhi(t, a.vecs_inverse)) : 0;
    const int vec = t - row * a.vecs;
    const Place at = at_row<ONE>(mine, row);
    const bool key = vec < a.Hkv;
    const int h = key ? vec : vec - a.Hkv;
    const int64_t from = key ? at.k : at.v;
    if (!in || !unit) continue;
    X8 y{};
    if (from >= 0) {
      const char* s = key ? a.c.k + from + h * a.c.k_head : a.c.v + from + h * a.c.v_head;
      if constexpr (KIND == kGather16) {
        y = *reinterpret_cast<const X8*>(s + u * 16);
      } else {
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(s + u * 4);
        RowCodec<4, false> codec;
        codec.load(reinterpret_cast<const uint8_t*>(s) + a.D / 2);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[e] = static_cast<T>(fp32_value(__builtin_fmaf(static_cast<float>((codes >> (4 * e)) & 15u), codec.scale, codec.bias)));
      }
    }
    char* d = a.out[key ? 0 : 1] + ((w.r0 + row) * a.Hkv + h) * a.D * 2 + u * 16;
    *reinterpret_cast<X8*>(d) = y;
  }
}

// Rows of few heads share a wave, so that its lanes have work; rows of many heads
// are shared out over waves while these do not fill the chip (eight waves a CU; all of
// them shared out: 94 for 65 us in the batch above).
void plan_rows(RowsArgs* a, int group) {
  const int64_t lanes = static_cast<int64_t>(a->vecs) * group;  // of a row
  a->tile_rows = 1;
  while (a->tile_rows < 64 && a->tile_rows * lanes < 128) a->tile_rows *= 2;
  a->vecs_inverse = a->vecs > 1 ? static_cast<uint32_t>(((1ull << 32) + a->vecs - 1) / a->vecs) : 0;
  const int64_t tiles = ceil_div(a->N, a->tile_rows), passes = ceil_div(a->tile_rows * lanes, 64);
  const int64_t most = ceil_div(static_cast<int64_t>(num_cus()) * 8, tiles);
  a->slices = static_cast<int32_t>(passes < most ? passes : most);
  a->waves = tiles * a->slices;
}

template <typename T, int GS, Kind KIND>
int launch_rows(const RowsArgs& a, hipStream_t s) {
  const int64_t blocks = ceil_div(a.waves, kRowsWaves);
  MX_REQUIRE(blocks < (1ll << 24), "too many rows: %lld", (long long)a.N);  // threads in 32 bits
  const dim3 grid(static_cast<unsigned>(blocks));
  if constexpr (KIND == kGather16 || KIND == kGather4) {
    if (a.tile_rows == 1) gather_kernel<T, GS, KIND, true><<<grid, kRowsWaves * 64, 0, s>>>(a);
    else gather_kernel<T, GS, KIND, false><<<grid, kRowsWaves * 64, 0, s>>>(a);
  } else {
    if (a.tile_rows == 1) rows_kernel<T, GS, KIND, true><<<grid, kRowsWaves * 64, 0, s>>>(a);
    else rows_kernel<T, GS, KIND, false><<<grid, kRowsWaves * 64, 0, s>>>(a);
  }
  MX_LAUNCH_CHECK();
  return MX_OK;
}

template <typename T, Kind KIND>
int rows_by_width(RowsArgs& a, hipStream_t s) {
  const int units = a.D / 8;
  const int group = units <= 4 ? 4 : units <= 8 ? 8 : 16;
  plan_rows(&a, group);
  if (group == 4) return launch_rows<T, 4, KIND>(a, s);
  if (group == 8) return launch_rows<T, 8, KIND>(a, s);
  return launch_rows<T, 16, KIND>(a, s);
}

template <Kind KIND>
int rows_by_type(RowsArgs& a, int32_t dtype, hipStream_t s) {
  return dtype == MX_DTYPE_BF16 ? rows_by_width<__bf16, KIND>(a, s) : rows_by_width<_Float16, KIND>(a, s);
}

int check_rows_operand(const mx_attention_tensor* t, const char* name) {
  MX_REQUIRE(t != nullptr && t->data != nullptr, "%s is null", name);
  MX_REQUIRE(reinterpret_cast<uintptr_t>(t->data) % 16 == 0 && t->row_stride % 8 == 0 && t->head_stride % 8 == 0 &&
                 t->row_stride >= 0 && t->head_stride >= 0,
             "%s: rows and heads must start at multiples of 16 bytes", name);
  return MX_OK;
}

int check_type(int32_t dtype, int32_t D) {
  MX_REQUIRE(dtype == MX_DTYPE_F16 || dtype == MX_DTYPE_BF16, "dtype %d is not fp16 or bf16", dtype);
  MX_REQUIRE(D > 0 && D % 8 == 0 && D <= MX_ATTENTION_MAX_D, "head width %d is no multiple of 8 up to %d", D,
             MX_ATTENTION_MAX_D);
  return MX_OK;
}

int check_rotary(const mx_rotary* r, int32_t D) {
  MX_REQUIRE(r->positions >= 0 && r->positions < (1ll << 31), "%lld positions", (long long)r->positions);
  MX_REQUIRE(r->pairs > 0 && r->pairs % 4 == 0 && 2 * r->pairs <= D,
             "%d pairs: twice their number must be a multiple of 8 up to the head width %d", r->pairs, D);
  MX_REQUIRE(r->positions == 0 || r->table != nullptr, "the rotary table is null");
  MX_REQUIRE(reinterpret_cast<uintptr_t>(r->table) % 16 == 0, "the rotary table must be 16-byte aligned");
  return MX_OK;
}

int set_lists(RowsArgs* a, int64_t N, int64_t B, const void* offsets, int32_t offsets_bytes, const void* starts,
              int32_t starts_bytes) {
  MX_REQUIRE(offsets != nullptr, "offsets are null");
  MX_REQUIRE((offsets_bytes == 4 || offsets_bytes == 8) && (starts == nullptr || starts_bytes == 4 || starts_bytes == 8),
             "index bytes %d and %d", offsets_bytes, starts_bytes);
  a->offsets = offsets, a->starts = starts;
  a->offsets_bytes = offsets_bytes, a->starts_bytes = starts_bytes;
  a->B = B, a->N = N;
  return MX_OK;
}

void set_source(RowsArgs* a, int i, const mx_attention_tensor* t) {
  a->src[i] = static_cast<const char*>(t->data);
  a->src_row[i] = t->row_stride * 2, a->src_head[i] = t->head_stride * 2;
}

void set_rotary(RowsArgs* a, const mx_rotary* r, float sign) {
  a->table = r->table, a->positions = r->positions;
  a->pairs = r->pairs, a->interleaved = r->interleaved, a->sign = sign;
}

}  // namespace
}  // namespace attn
}  // namespace mx

extern "C" int mx_jagged_rotary(int32_t dtype, const mx_attention_tensor* x, int64_t N, int32_t H, int32_t D,
                                const mx_rotary* rotary, int32_t inverse, int64_t B, const void* offsets,
                                int32_t offsets_bytes, const void* starts, int32_t starts_bytes, void* out,
                                void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_type(dtype, D)) return rc;
  MX_REQUIRE(N >= 0 && B >= 0 && H >= 0 && H < (1 << 20), "bad sizes");
  MX_REQUIRE(rotary != nullptr, "rotary is null");
  if (int rc = check_rotary(rotary, D)) return rc;
  if (N == 0 || H == 0) return MX_OK;
  if (int rc = check_rows_operand(x, "x")) return rc;
  MX_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0, "out is null or not 16-byte aligned");
  RowsArgs a{};
  if (int rc = set_lists(&a, N, B, offsets, offsets_bytes, starts, starts_bytes)) return rc;
  set_source(&a, 0, x);
  set_rotary(&a, rotary, inverse ? -1.0f : 1.0f);
  a.out[0] = static_cast<char*>(out);
  a.H = H, a.Hkv = 0, a.D = D, a.vecs = H;
  return rows_by_type<kRotate>(a, dtype, mx::as_stream(stream));
}

extern "C" int mx_paged_cache_append_rows(const mx_paged_cache* cache, int32_t bits, int32_t dtype, int32_t H,
                                          int32_t Hkv, int32_t D, const mx_attention_tensor* q,
                                          const mx_attention_tensor* k, const mx_attention_tensor* v,
                                          const mx_rotary* rotary, int64_t N, int64_t B, const void* offsets,
                                          int32_t offsets_bytes, const void* starts, int32_t starts_bytes,
                                          void* q_out, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_rows_cache(cache, bits)) return rc;
  if (int rc = check_type(dtype, D)) return rc;
  MX_REQUIRE(N >= 0 && B >= 0 && H >= 0 && H < (1 << 20) && Hkv > 0 && Hkv < (1 << 20), "bad sizes");
  MX_REQUIRE(H == 0 || rotary != nullptr, "queries without a rotation");
  if (rotary != nullptr)
    if (int rc = check_rotary(rotary, D)) return rc;
  if (N == 0) return MX_OK;
  if (int rc = check_rows_operand(k, "k")) return rc;
  if (int rc = check_rows_operand(v, "v")) return rc;
  MX_REQUIRE(B == 0 || starts != nullptr, "starts are null");
  MX_REQUIRE(cache->table != nullptr || cache->table_width == 0 || B == 0, "the page table is null");
  RowsArgs a{};
  if (int rc = set_lists(&a, N, B, offsets, offsets_bytes, starts, starts_bytes)) return rc;
  if (H > 0) {
    if (int rc = check_rows_operand(q, "q")) return rc;
    MX_REQUIRE(q_out != nullptr && reinterpret_cast<uintptr_t>(q_out) % 16 == 0, "q_out is null or not 16-byte aligned");
    set_source(&a, 0, q);
    a.out[0] = static_cast<char*>(q_out);
  }
  set_source(&a, 1, k);
  set_source(&a, 2, v);
  if (rotary != nullptr) set_rotary(&a, rotary, 1.0f);
  a.c = cache_of(cache, bits == 16 ? 2 : 1);
  a.H = H, a.Hkv = Hkv, a.D = D, a.vecs = H + 2 * Hkv;
  const hipStream_t s = mx::as_stream(stream);
  return bits == 16 ? rows_by_type<kAppend16>(a, dtype, s) : rows_by_type<kAppend4>(a, dtype, s);
}

extern "C" int mx_paged_cache_gather(const mx_paged_cache* cache, int32_t bits, int32_t dtype, int32_t Hkv, int32_t D,
                                     int64_t N, int64_t B, const void* offsets, int32_t offsets_bytes, void* k_out,
                                     void* v_out, void* stream) {
  using namespace mx::attn;
  mx::clear_error();
  if (int rc = check_rows_cache(cache, bits)) return rc;
  if (int rc = check_type(dtype, D)) return rc;
  MX_REQUIRE(N >= 0 && B >= 0 && Hkv > 0 && Hkv < (1 << 20), "bad sizes");
  if (N == 0) return MX_OK;
  MX_REQUIRE(k_out != nullptr && v_out != nullptr && reinterpret_cast<uintptr_t>(k_out) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(v_out) % 16 == 0,
             "outputs are null or not 16-byte aligned");
  MX_REQUIRE(cache->table != nullptr || cache->table_width == 0 || B == 0, "the page table is null");
  RowsArgs a{};
  if (int rc = set_lists(&a, N, B, offsets, offsets_bytes, nullptr, 0)) return rc;
  a.out[0] = static_cast<char*>(k_out), a.out[1] = static_cast<char*>(v_out);
  a.c = cache_of(cache, bits == 16 ? 2 : 1);
  a.Hkv = Hkv, a.D = D, a.vecs = 2 * Hkv;
  const hipStream_t s = mx::as_stream(stream);
  return bits == 16 ? rows_by_type<kGather16>(a, dtype, s) : rows_by_type<kGather4>(a, dtype, s);
}
