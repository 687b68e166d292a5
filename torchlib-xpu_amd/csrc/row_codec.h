// The scale and bias of a quantized row, and one element's code: what the codec
// ops and the 4-bit key-value cache share.
#pragma once

#include "mx_common.h"

namespace mx {
namespace {

__device__ __forceinline__ float round_to_half(float v) { return __half2float(__float2half_rn(v)); }

// A row's codec: scale and bias from its range, one element's code, and the
// scale and bias as the row ends with them.  BITS 8 with FUSED8: the 8-bit
// format (fp32 scale and bias); else the N-bit format (fp16).
template <int BITS, bool FUSED8>
struct RowCodec {
  static constexpr int kTail = FUSED8 ? 8 : 4;  // bytes after the codes
  static constexpr int kMax = (1 << BITS) - 1;
  float scale, bias, inv;
  __device__ __forceinline__ void set(float mn, float mx) {
    if constexpr (FUSED8) {
      const float range = mx - mn;
      scale = range / 255.0f;
      inv = 255.0f / (range + 1e-8f);
      bias = mn;
    } else {
      bias = round_to_half(mn);
      const float range = mx - bias;
      scale = range == 0.0f ? 1.0f : range / static_cast<float>(kMax);
      scale = round_to_half(scale);
      if (scale == 0.0f) scale = 1.0f;  // underflow in fp16
      inv = 1.0f / scale;
      if (__builtin_isinf(inv)) {
        scale = 1.0f;
        inv = 1.0f;
      }
    }
  }
  __device__ __forceinline__ uint32_t code(float x) const {
    float q = __builtin_rintf(__fmul_rn(x - bias, inv));
    if constexpr (FUSED8) return static_cast<uint8_t>(q);
    q = q > 0.0f ? (q > static_cast<float>(kMax) ? static_cast<float>(kMax) : q) : 0.0f;  // NaN: 0
    return static_cast<uint32_t>(q);
  }
  __device__ __forceinline__ void store(uint8_t* o) const {
    if constexpr (FUSED8) {
      __builtin_memcpy(o, &scale, 4);
      __builtin_memcpy(o + 4, &bias, 4);
    } else {
      const __half hs = __float2half_rn(scale), hb = __float2half_rn(bias);
      const uint32_t w = static_cast<uint32_t>(__half_as_ushort(hs)) |
                         (static_cast<uint32_t>(__half_as_ushort(hb)) << 16);
      __builtin_memcpy(o, &w, 4);
    }
  }
  __device__ __forceinline__ void load(const uint8_t* x) {
    if constexpr (FUSED8) {
      __builtin_memcpy(&scale, x, 4);
      __builtin_memcpy(&bias, x + 4, 4);
    } else {
      uint32_t w;
      __builtin_memcpy(&w, x, 4);
      scale = __half2float(__ushort_as_half(static_cast<uint16_t>(w & 0xffffu)));
      bias = __half2float(__ushort_as_half(static_cast<uint16_t>(w >> 16)));
    }
  }
};

}  // namespace
}  // namespace mx
