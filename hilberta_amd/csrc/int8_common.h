// 16-bit values to 8-bit whole numbers by their row's largest, as the row kernels and the products of a few rows
// need them.
//
// Of 16-bit rows q is exact.  A value is a 2^i and the top b 2^j, i <= j, with a, b < 2^11 (fp16's significand;
// bf16's has 8 bits): the quotient 127 x / top = 127 a / (b 2^(j - i)) is off a tie, k + 1/2, by |254 a - (2k + 1)
// b 2^(j - i)| / (2 b 2^(j - i)), a whole number over that: nothing, and the tie comes out as itself, or at least 1
// / (254 a) > 2^-19 of the quotient, far more than its fp32 error.  127 x itself, of 18 bits at most, is exact in
// fp32.  Rows of fp32 values (the AdaLN pass) have no such margin: there a quotient within fp32's error of a tie
// may go either way.
//
// The largest value is found on the bit patterns without the sign, in which an infinity is above every number and a
// NaN above that.
#pragma once
#include "common.h"

namespace hb {
namespace {

constexpr int MAX_FEATURES = 1 << 17;  // 2^17 x 127 x 128 < 2^31: the product's sums stay in 32 bits

// What turns a row's values into whole numbers: q = rint(127 x / top).
struct Scaler {
  float top, inverse, factor, scale;
  // bits: the largest pattern of |x| as fp32.
  __device__ explicit Scaler(uint32_t bits) {
    const float t = __builtin_bit_cast(float, bits);
    const bool finite = bits < 0x7f800000u;
    // (reciprocals of the smallest tops and 127 times the largest would overflow: rows out there are taken
    // 2^64 times as large, or as small)
    const float up = t < 0x1p-60f ? 0x1p64f : t > 0x1p60f ? 0x1p-64f : 1.f;
    scale = finite ? t / 127.f : __builtin_nanf("");
    const bool zero = !finite || bits == 0;
    top = t * up;
    inverse = zero ? 0.f : __builtin_amdgcn_rcpf(top);
    top = zero ? 0.f : top;
    factor = zero ? 0.f : 127.f * up;
  }
  // The whole number, in the low byte.  The quotient as the reciprocal gives it, and one correction by its
  // remainder, which an fma gives exactly: a quotient that fits 24 bits, as every tie does, comes out as
  // itself.  Adding 1.5 x 2^23 rounds it to even, in the lowest bits of the sum.
  __device__ uint32_t quantize(float x) const {
    const float t = x * factor;
    const float y = t * inverse;
    return __builtin_bit_cast(uint32_t, __builtin_fmaf(__builtin_fmaf(-y, top, t), inverse, y) + 12582912.f);
  }
};

// The low bytes of a, b, c and d.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400), __builtin_amdgcn_perm(b, a, 0x0c0c0400), 0x05040100);
}

__device__ __forceinline__ u32x2 pack_row8(const Scaler& s, const float (&x)[8]) {
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = s.quantize(x[i]);
  return u32x2{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7])};
}

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

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The larger patterns of |x|, pair by pair.
__device__ __forceinline__ u16x2 max_pairs(u16x2 top, const u32x4& raw) {
#pragma unroll
  for (int k = 0; k < 4; ++k) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, raw[k] & 0x7fff7fffu));
  return top;
}

// The fp32 bits of the larger of two 16-bit values.
template <bool F16>
__device__ __forceinline__ uint32_t fp32_bits(u16x2 top) {
  return __builtin_bit_cast(uint32_t, to_f<F16>(top[0] > top[1] ? top[0] : top[1]));
}

}  // namespace
}  // namespace hb
