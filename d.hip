#include <hip/hip_runtime.h>
#include <cstdint>
__global__ void k16(const int64_t* in, int64_t width, int64_t* out) {
  const int64_t start = in[0], off = in[1], row = blockIdx.x;
  const int64_t t = start + row - off;
  if (start < 0 || t < 0) return;
  const int64_t e = t >> 4;
  if (e >= width) return;
  out[0] = e;
}
