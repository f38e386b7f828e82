// What the products of 8-bit and 16-bit rows share: direct loads to LDS and their waits, the walk over output tiles,
// and the stages of a ring known at compile time.
#pragma once
#include <type_traits>
#include <utility>

#include "common.h"

namespace hb {
namespace {

__device__ __forceinline__ float gelu(float v) {
  // v (1 + tanh u) / 2 = v / (1 + exp(-2u)),  u = sqrt(2 / pi) (v + 0.044715 v^3);  -2u / ln 2 by its powers
  const float e = v * (-2.302208198144325f - 0.1029432395800235f * v * v);
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e));
}

typedef __attribute__((address_space(3))) void* lds_ptr;

// word 3 of a raw buffer resource (32-bit data format, no swizzle)
constexpr int BUFFER_WORD3 = 0x00020000;

// 16 bytes a lane from base + voffset + soffset into LDS at dst + 16 lane.  (The buffer resource type exists
// for the device target only; the host pass sees an empty body.)
__device__ __forceinline__ void load_lds16(const void* base, void* dst, int voffset, int soffset) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, BUFFER_WORD3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)dst, 16, voffset, soffset, 0, 0);
#endif
}

// s_waitcnt vmcnt(N): all but the last N loads have arrived.
template <int N>
__device__ __forceinline__ void wait_arrivals() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0f70);
}

// The same, and this wave's reads of LDS.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);
}

// A barrier that no access to LDS is moved across.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A value of another of 16 neighbouring lanes.
template <int CONTROL>
__device__ __forceinline__ uint32_t moved_bits(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true);
}
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, moved_bits<CONTROL>(__builtin_bit_cast(uint32_t, v)));
}
// The sum over 16 neighbouring lanes, in each of them: of pairs, of quads, of the mirrored half row and row.
__device__ __forceinline__ float sum16(float v) {
  v += moved<0xb1>(v);
  v += moved<0x4e>(v);
  v += moved<0x141>(v);
  return v + moved<0x140>(v);
}

template <typename Begin, int... I>
__device__ __forceinline__ void begin_all(Begin& begin, std::integer_sequence<int, I...>) {
  (begin(std::integral_constant<int, I>()), ...);
}
// Whether one of the steps was the last.
template <typename Step, int... I>
__device__ __forceinline__ bool step_all(Step& step, std::integer_sequence<int, I...>) {
  return (step(std::integral_constant<int, I>()) || ...);
}

// Which tile a workgroup takes.
struct Tile {
  int set, c0;
  uint32_t t0;
};

// Tiles walk bands of `BAND` token tiles, channel tile by channel tile.
template <int TC, int TT, int BAND, typename Args>
__device__ __forceinline__ Tile tile_at(const Args& a, uint32_t tile) {
  const int set = tile >= a.tiles0;
  if (set) tile -= a.tiles0;
  const uint32_t token_tiles = (a.set[set].tokens + TT - 1) / TT;
  const uint32_t band = tile / (BAND * a.channel_tiles), in_band = tile - band * (BAND * a.channel_tiles);
  const uint32_t height = min((uint32_t)BAND, token_tiles - band * BAND);
  const uint32_t c = in_band / height;
  return {set, (int)c * TC, (band * BAND + in_band - c * height) * TT};
}

__device__ __forceinline__ const int8_t* uniform_pointer(const int8_t* p) {
  const uint64_t v = (uint64_t)p;
  return (const int8_t*)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

}  // namespace
}  // namespace hb
