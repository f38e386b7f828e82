// Rows of 16-bit values at any address and of any length, eight values at a time.
#pragma once
#include "common.h"

namespace hb {
namespace {

// (the hardware takes 16 bytes from any 2-byte address)
typedef u32x4 __attribute__((aligned(2))) any_u32x4;

// `raw` without its first `n` values, zeros after the others.
__device__ __forceinline__ u32x4 drop_values(const u32x4& raw, int n) {
  uint64_t lo = raw[0] | (uint64_t)raw[1] << 32, hi = raw[2] | (uint64_t)raw[3] << 32;
  if (n >= 4) lo = hi, hi = 0, n -= 4;
  if (n >= 4) lo = 0, n = 0;
  if (n) lo = lo >> (16 * n) | hi << (64 - 16 * n), hi >>= 16 * n;
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// Values col .. col + 7 of a row as stored, zeros past the row: the last ones come with those before them.
template <bool STREAM>
__device__ __forceinline__ u32x4 load_row8(const uint16_t* row, int col, int features) {
  u32x4 raw = {0, 0, 0, 0};
  if (features >= 8) {
    const int at = min(col, features - 8);
    if (col < features) {
      if constexpr (STREAM) raw = __builtin_nontemporal_load((const any_u32x4*)(row + at));
      else raw = *(const any_u32x4*)(row + at);
    }
    if (col > at) raw = drop_values(raw, min(col - at, 8));
  } else if (col == 0) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < features) raw[i >> 1] |= (uint32_t)row[i] << (16 * (i & 1));
  }
  return raw;
}

}  // namespace
}  // namespace hb
