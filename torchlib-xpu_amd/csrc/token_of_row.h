// The token of its sequence that a packed row is.  Plain C++, host and device.
#pragma once

#include <cstdint>

namespace mx {
namespace attn {

// A list's row at `offset` is its sequence's token `start`: row `row` is token
// start + (row - offset), or -1 (none) where start is negative, the row lies before
// the list, or the sum does not fit 63 bits.  start and offset may hold
// anything: in signed arithmetic the compiler would take it that sums of
// numbers found not negative are not negative either, and drop that check.
constexpr int64_t token_of_row(int64_t start, int64_t row, int64_t offset) {
  if (start < 0 || offset > row) return -1;
  const uint64_t most = INT64_MAX;
  const uint64_t i = static_cast<uint64_t>(row) - static_cast<uint64_t>(offset);
  const uint64_t t = static_cast<uint64_t>(start) + i;  // below 2^64 for i <= most
  return i <= most && t <= most ? static_cast<int64_t>(t) : -1;
}

}  // namespace attn
}  // namespace mx
