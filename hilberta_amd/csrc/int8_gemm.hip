// Products of 8-bit rows with an 8-bit weight: the linear layers of the denoiser's blocks, and their Q/K/V
// projection with the heads' RMSNorm and the position rotation in the same pass.
//
//   p[m, n] = (sum_k q[m, k] w[n, k]) * scale[m] * weight_scale[n] + bias[n]
//   linear:  out = p, or GELU(tanh)(p)
//   qkv:     channels n are [Q | K | V] of `heads` heads of 128;  Q and K: p * rsqrt(mean p^2 + eps) * norm
//            over each head, pairs (2i, 2i + 1) turned by the token's cos and sin;  V: p
//
// The sums are whole numbers in 32 bits, exact in any order; everything after them is fp32 and is rounded
// once, to the 16-bit output.
//
// The weight's channels are the rows of the matrix instruction (v_mfma_i32_32x32x32_i8) and the tokens its
// columns: a lane then holds one token's values, 4 consecutive channels an accumulator quarter, so that they move
// 16 bytes at a time and a token's scale is one register.
//
// Three kernels: many rows (int8_wide_kernel), fewer (int8_tile_kernel), and a few that come in 16 bits and are
// quantized in the same launch (int8_few_kernel, linear only).
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "int8_common.h"
#include "../../include/hilberta_hip.h"

namespace hb {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int HEAD = 128;

// One set of rows with its weight.  Two sets (a block's text and image rows) share a launch.
struct Set {
  const int8_t* q;          // [tokens, padded]
  const float* scale;       // [tokens]
  const int8_t* w;          // [columns, padded]
  const float* w_scale;     // [columns]
  const uint16_t* bias;     // [columns] or null
  uint16_t* out;            // qkv: where this set's first token goes
  const uint16_t* norm[2];  // qkv: weights of Q's and K's heads [128], or null
  int64_t out_b, out_n;     // output strides of a batch element and a row
  uint32_t rows, tokens;    // rows of a batch element, and of all
  uint32_t first;           // qkv: the first row's place in cos and sin
  uint32_t start;           // rows of the set before these (which another launch takes)
};

struct Args {
  Set set[2];
  int32_t columns, padded;
  uint32_t tiles0, tiles, tiles_xcd;  // tiles of set 0, of all, and of an XCD
  uint32_t channel_tiles;             // tiles along the channels
  int32_t gelu, vectors;           // vectors: every output row takes 16-byte stores
  const float* cos;                // qkv: [rows of both sets, 128] or null
  const float* sin;
  int64_t out_p;                   // qkv: output stride of Q, K and V
  int32_t heads;
  float eps;
};

__device__ __forceinline__ float gelu(float v) {
  // v (1 + tanh u) / 2 = v / (1 + exp(-2u)),  u = sqrt(2 / pi) (v + 0.044715 v^3);  -2u / ln 2 by its powers
  const float e = v * (-2.302208198144325f - 0.1029432395800235f * v * v);
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e));
}

// Four values of this lane's token, channels c .. c + 3 with c = 8g + 4 (lane / 32), of quarters g = 2p
// (`even`) and 2p + 1 (`odd`) of a 32-channel accumulator, to 16 bits and exchanged with the other half of
// the wave: lanes below 32 then hold channels 16p .. 16p + 7 of their token, the others 16p + 8 .. 16p + 15.
template <bool F16>
__device__ __forceinline__ u32x4 pack_pair(const float (&even)[4], const float (&odd)[4]) {
  auto two = [](float a, float b) { return (uint32_t)from_f<F16>(a) | (uint32_t)from_f<F16>(b) << 16; };
  const auto lo = __builtin_amdgcn_permlane32_swap(two(even[0], even[1]), two(odd[0], odd[1]), false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap(two(even[2], even[3]), two(odd[2], odd[3]), false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
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

// ------------------------------------------------------------------ what every kernel does with its sums
// The epilogue's values of a tile's channels, in LDS: weight scale, bias, head norm.
template <bool F16, bool QKV, int TC>
__device__ __forceinline__ void load_channels(const Args& a, const Set& s, int c0, float (&channel)[3][TC]) {
  const int i = threadIdx.x;
  if (i >= TC) return;
  const int c = min(c0 + i, a.columns - 1);
  const int plane = QKV ? c / (a.heads * HEAD) : 2;
  channel[0][i] = s.w_scale[c];
  channel[1][i] = s.bias ? to_f<F16>(s.bias[c]) : 0.f;
  channel[2][i] = QKV && plane < 2 && s.norm[plane] ? to_f<F16>(s.norm[plane][i & (HEAD - 1)]) : 1.f;
}

// Token `at` of a set (clamped to its last): where it goes, in elements from s.out, and where its row of the
// rotary tables begins.
__device__ __forceinline__ int64_t row_of(const Set& s, uint32_t at) {
  const uint32_t token = s.start + min(at, s.tokens - 1), b = token / s.rows;
  return b * s.out_b + (int64_t)(token - b * s.rows) * s.out_n;
}
__device__ __forceinline__ int64_t table_of(const Set& s, uint32_t at) {
  return (int64_t)(s.first + (s.start + min(at, s.tokens - 1)) % s.rows) * HEAD;
}

// Eight values of channels c .. c + 7 to `out`, those of them that there are.
template <bool QKV>
__device__ __forceinline__ void store8(const Args& a, uint16_t* out, int c, const u32x4& v) {
  typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint32_t words3 __attribute__((ext_vector_type(3), aligned(4)));
  if (QKV ? c < a.columns : c + 8 <= a.columns) {
    if (QKV || a.vectors) {
      __builtin_nontemporal_store(v, (u32x4*)out);
    } else if ((uintptr_t)out & 2) {
      out[0] = (uint16_t)v[0];
      *(words3*)(out + 1) = words3{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16};
      out[7] = (uint16_t)(v[3] >> 16);
    } else {
      *(words4*)out = v;
    }
  } else if (!QKV) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < a.columns) out[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
  }
}

// The sum over 16 neighbouring lanes, in each of them: of pairs, of quads, of the mirrored half row and row.
template <int CONTROL>
__device__ __forceinline__ uint32_t moved_bits(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true);
}
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, moved_bits<CONTROL>(__builtin_bit_cast(uint32_t, v)));
}
__device__ __forceinline__ float sum16(float v) {
  v += moved<0xb1>(v);
  v += moved<0x4e>(v);
  v += moved<0x141>(v);
  return v + moved<0x140>(v);
}

// Two pairs (2i, 2i + 1) turned by cos and sin.
__device__ __forceinline__ void rotate(float* v, const f32x4& cos, const f32x4& sin) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const float even = v[k], odd = v[k + 1];
    v[k] = even * cos[k] - odd * sin[k];
    v[k + 1] = odd * cos[k + 1] + even * sin[k + 1];
  }
}

// The epilogue of a wave's 32 tokens from t0 on and 32 CF channels from c0 on (linear); `channel` are those
// channels' values, TC apart.  Lanes l and l + 32 hold token t0 + l % 32.  After pack_pair a 32-channel block of
// a token is four 16-byte chunks, two in each of those lanes; exchanged with the lane 16 on, four lanes hold a
// token's four chunks, and a store writes 64 bytes a row (32 without: 16896 x 3072 x 12288 586 -> 580 us).
//
// Stores of 16 bytes, here and below, bypass the caches at every size, which leaves those to the operands.  Measured
// alone and with int8_rows reading the output next, us past the caches / through them: 16384 x 3072 x 12288 with GELU
// (403 MB) 555, 665 / 584, 680; 8192 rows 286, 328 / 292, 335; 16384 x 3072 x 3072 (101 MB) 149, 182 / 162, 181; 4096
// rows 46, 54.6 / 46, 54.4; 512 x 3072 x 12288 (13 MB) 39.6, 45.2 / 40.6, 45.6; 77 x 4096 x 3072 8.1, 11.9 / 8.1, 11.6;
// qkv of 512 + 16384 tokens 476, 554 / 494, 555, of 512 + 1024 57.5, 63.3 / 56.3, 64.3.  Where it loses is one row that
// is read next: 1 x 3072 x 18432 13.7, 22.9 / 13.9, 21.2.
template <bool F16, bool GELU, int CF, int TC>
__device__ __forceinline__ void finish(const Args& a, const Set& s, const i32x16 (&acc)[CF], float scale,
                                       const float* channel, int c0, uint32_t t0) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int chunk = (lane >> 4 & 1) * 2 + half;
  uint16_t* out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) out[h] = s.out + row_of(s, t0 + h * 16 + (lane & 15)) + c0 + chunk * 8;
  channel += half * 4;
#pragma unroll
  for (int i = 0; i < CF; ++i) {
    u32x4 packed[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float v[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int c = i * 32 + (2 * p + g) * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float y = (float)acc[i][8 * p + 4 * g + k] * scale * channel[c + k] + channel[TC + c + k];
          v[g][k] = GELU ? gelu(y) : y;
        }
      }
      packed[p] = pack_pair<F16>(v[0], v[1]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const auto both = __builtin_amdgcn_permlane16_swap(packed[0][k], packed[1][k], false, false);
      packed[0][k] = both[0];
      packed[1][k] = both[1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (t0 + h * 16 + (lane & 15) < s.tokens) store8<false>(a, out[h] + i * 32, c0 + i * 32 + chunk * 8, packed[h]);
    __builtin_amdgcn_sched_barrier(0);  // (a block at a time: all at once take more registers than there are)
  }
}

// Channels c0 + c .. + 7 of token `at`, of its sums and scale (qkv: 16 neighbouring lanes hold a head).
template <bool F16, bool QKV, bool GELU, int TC>
__device__ __forceinline__ void finish8(const Args& a, const Set& s, const i32x4 (&sum)[2], float scale,
                                        const float (&channel)[3][TC], int c0, uint32_t at, int c) {
  const int plane = QKV ? c0 / (a.heads * HEAD) : 2;
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (float)sum[k >> 2][k & 3] * scale * channel[0][c + k] + channel[1][c + k];
  uint16_t* out = s.out + row_of(s, at) + c0 + c;
  if (QKV) {
    out += plane * a.out_p - plane * a.heads * HEAD;
    if (plane < 2) {
      float squares = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) squares += v[k] * v[k];
      const float rms = __builtin_amdgcn_rsqf(sum16(squares) * (1.f / HEAD) + a.eps);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= rms * channel[2][c + k];
      const int64_t table = table_of(s, at) + c;
      if (a.cos) {
#pragma unroll
        for (int g = 0; g < 8; g += 4)
          rotate(v + g, *(const f32x4*)(a.cos + table + g), *(const f32x4*)(a.sin + table + g));
      }
    }
  } else if (GELU) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = gelu(v[k]);
  }
  if (at < s.tokens) store8<QKV>(a, out, c0 + c, pack8<F16>(v));
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

// The epilogue of a wave's 32 tokens from t0 on and one head from c0 on (qkv).  Lanes l and l + 32 hold token
// t0 + l % 32, and would read its rotary rows and write its output 32 bytes at a time.  So 16 tokens at a time go
// through the wave's own part of a stage, eight pieces of 1 KB, and come back as four tokens of 16 lanes each,
// whose reads and writes are whole lines (512 + 16384 rows x 3072, 24 heads: 511 -> 479 us).  `channel` are the head's values, TC apart.
template <bool F16, bool TURN, int TC>
__device__ __forceinline__ void finish_head(const Args& a, const Set& s, const i32x16 (&acc)[4], float scale,
                                            const float* channel, int c0, uint32_t t0, int8_t* box) {
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, c = (lane & 15) * 8;
  const int plane = c0 / (a.heads * HEAD);
  const bool heads = TURN || plane < 2, one = s.start + s.tokens <= s.rows;  // (one batch element: no division)
  uint16_t* const out = s.out + plane * a.out_p + (c0 - plane * a.heads * HEAD) + c;
  auto place = [&](int token) { return (token >> 1) * 8192 + (token & 1) * 512; };
  float ws[8], bias[8], norm[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) ws[k] = channel[c + k], bias[k] = channel[TC + c + k], norm[k] = channel[2 * TC + c + k];
  // Four tokens' places, and their rotary values, asked for four tokens ahead.
  struct Ahead {
    uint32_t at;
    int64_t row;
    f32x4 cos[2], sin[2];
  };
  auto ask = [&](int m) {
    Ahead to;
    to.at = t0 + m * 4 + (lane >> 4);
    uint32_t n = s.start + min(to.at, s.tokens - 1), b = 0;
    if (!one) b = n / s.rows, n -= b * s.rows;
    to.row = b * s.out_b + (int64_t)n * s.out_n;
    if (TURN) {
      const int64_t table = (int64_t)(s.first + n) * HEAD + c;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        to.cos[g] = *(const f32x4*)(a.cos + table + g * 4);
        to.sin[g] = *(const f32x4*)(a.sin + table + g * 4);
      }
    }
    return to;
  };
  Ahead next = ask(0);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (col >> 4 == p) {
      int token = lane & 15;
      asm volatile("" : "+v"(token));  // (or the addresses stay in registers from here to the next tile)
      int8_t* const to = box + place(token);
      // (units of four channels, in an order of the token's, so that tokens' lie in different banks)
      const int order = token ^ half;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(i32x4*)(to + (((i & 1) * 8 + g * 2) ^ order) * 16 + (i >> 1) * 256) =
              i32x4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      const Ahead now = next;
      const int token = q * 4 + (lane >> 4);
      next = ask(p * 4 + q + 1);
      const float token_scale = __shfl(scale, p * 16 + token, 64);
      i32x4 sum[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) sum[g] = *(const i32x4*)(box + place(token) + (c / 4 + g ^ token) * 16);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (float)sum[k >> 2][k & 3] * token_scale * ws[k] + bias[k];
      if (heads) {
        float squares = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) squares += v[k] * v[k];
        const float rms = __builtin_amdgcn_rsqf(sum16(squares) * (1.f / HEAD) + a.eps);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= rms * norm[k];
        if (TURN) {
#pragma unroll
          for (int g = 0; g < 2; ++g) rotate(v + 4 * g, now.cos[g], now.sin[g]);
        }
      }
      if (now.at < s.tokens) __builtin_nontemporal_store(pack8<F16>(v), (u32x4*)(out + now.row));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Which tile a workgroup takes.
struct Tile {
  int set, c0;
  uint32_t t0;
};

// Tiles walk bands of `BAND` token tiles, channel tile by channel tile.
template <int TC, int TT, int BAND>
__device__ __forceinline__ Tile tile_at(const Args& a, uint32_t tile) {
  const int set = tile >= a.tiles0;
  if (set) tile -= a.tiles0;
  const uint32_t token_tiles = (a.set[set].tokens + TT - 1) / TT;
  const uint32_t band = tile / (BAND * a.channel_tiles), in_band = tile - band * (BAND * a.channel_tiles);
  const uint32_t height = min((uint32_t)BAND, token_tiles - band * BAND);
  const uint32_t c = in_band / height;
  return {set, (int)c * TC, (band * BAND + in_band - c * height) * TT};
}

// Where rows end.  A stage is 128 features, and rows a multiple of 64: what a lane's load asks for past the row
// (its chunk of a last half stage, or a stage after the last) is moved outside the buffer, from where a load
// brings zeros and reads nothing.
struct Ends {
  int full, beyond;  // whole stages, and what the stage after them adds to this lane's offset
  __device__ Ends(int padded, int chunk)
      : full(padded >> 7), beyond((padded & 64) && chunk < 4 ? 0 : (int)0x80000000) {}
  __device__ int past(int stage) const {
    return stage < full ? 0 : stage == full ? beyond : (int)0x80000000;
  }
};

// ------------------------------------------------------------------ many rows
// 256 channels x 256 tokens a workgroup of eight waves, 128 x 64 each; one workgroup a CU, which walks its
// tiles.  Bound by the loads: the same kernel without them runs at 3.0 POP/s, with them at 2.45 (16384 x 12288 x
// 3072 in 504 us).  So the tile is as large as the registers allow (128 x 256 tiles, two workgroups a CU, move half
// as much again: 620 us), and a stage is 128 features deep: a row's 128 bytes are one request to the L2 (64-byte
// rows, twice as many requests, took the smaller tiles from 2.4 to 1.9 POP/s).
//  * Two stages of 64 KB in LDS, by direct loads, spread among the products (asked for together they hold up the
//    products' issue): half of stage n + 2 while the last step of stage n is multiplied, which everyone has read
//    by then, the other half with the first step of n + 1.
//  * The operands of a 32-feature step are read while the step before multiplies; the scheduler is held to
//    that order (left alone it reads them just before their use: 2.25 instead of 2.44 POP/s).
//  * A tile's last stage asks for the first stages of the next, which the epilogue then hides (qkv: for the
//    first only, since its epilogue works in the second's place).
//  * An XCD takes a run of the tiles, four token tiles by all channel tiles at a time (bands of 8 token tiles:
//    16896 x 3072 x 12288 630 us, of 4: 586), so that its L2 serves both operands.
constexpr int WIDE = 256, WIDE_STEP = 128, WIDE_BAND = 4;
constexpr int WIDE_STAGE = 2 * WIDE * WIDE_STEP;     // 64 KB
constexpr int WIDE_LOADS = WIDE_STAGE / 1024 / 8;    // 1 KB loads of a wave and stage

__device__ __forceinline__ const int8_t* uniform_pointer(const int8_t* p) {
  const uint64_t v = (uint64_t)p;
  return (const int8_t*)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

template <bool F16, bool QKV, bool GELU>
__global__ __launch_bounds__(512, 2) void int8_wide_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) int8_t lds0[WIDE_STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds1[WIDE_STAGE];
  __shared__ __attribute__((aligned(16))) float channel[2][3][WIDE];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int wc = wave & 1, wt = wave >> 1;
  const int stages = (a.padded + 2 * WIDE_STEP - 1) / (2 * WIDE_STEP) * 2;  // (an even number)
  // (workgroups go to the eight XCDs in turn)
  const uint32_t first = (blockIdx.x & 7) * a.tiles_xcd, stride = gridDim.x >> 3;
  uint32_t slot = blockIdx.x >> 3;
  if (slot >= a.tiles_xcd || first + slot >= a.tiles) return;
  // Loads: a wave's load j fills LDS rows 8 (8 j + wave) .. + 7, eight lanes a row; rows below WIDE are
  // channels, the others tokens (rows past the operands' ends: the last ones again).  The lane at slot p of
  // row r loads chunk p ^ (r / 2 % 8), so that the chunks that 16 rows' lanes read together lie in
  // different banks.
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  const Ends ends(a.padded, chunk);
  const int8_t *wbase, *qbase;
  int offset[WIDE_LOADS];
  auto aim = [&](const Tile& t) {
    const Set& s = a.set[t.set];
    wbase = uniform_pointer(s.w + (int64_t)t.c0 * a.padded);
    qbase = uniform_pointer(s.q + (int64_t)t.t0 * a.padded);
#pragma unroll
    for (int j = 0; j < WIDE_LOADS; ++j) {
      const int r = 8 * (8 * j + wave) + (lane >> 3);
      const int row = 64 * j < WIDE ? min(r, a.columns - 1 - t.c0) : (int)min((uint32_t)(r - WIDE), s.tokens - 1 - t.t0);
      offset[j] = row * a.padded + chunk * 16;
    }
  };
  auto load = [&](int8_t* dst, int stage, int j, int past) {
    load_lds16(64 * j < WIDE ? wbase : qbase, dst + 1024 * (8 * j + wave), offset[j] | past, uniform(stage * WIDE_STEP));
  };
  // Operands: lane l holds bytes 16 (l / 32) .. + 15 of a 32-byte step of row l % 32.
  const int read = col * WIDE_STEP + ((col >> 1 & 7) ^ half) * 16;
  i32x4 w[2][4], x[2][2];
  auto fetch = [&](const int8_t* src, int u) {
    const int at = read ^ (u * 32);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[u & 1][i] = *(const i32x4*)(src + (wc * 128 + i * 32) * WIDE_STEP + at);
#pragma unroll
    for (int j = 0; j < 2; ++j) x[u & 1][j] = *(const i32x4*)(src + (WIDE + wt * 64 + j * 32) * WIDE_STEP + at);
  };
  i32x16 acc[2][4];
  auto pin = [] { __builtin_amdgcn_sched_barrier(0); };
  // Eight products, with loads `from` .. `from` + 3 of a stage to `dst` among them.
  auto products = [&](auto loads, int u, int8_t* dst, int stage, int from) {
    constexpr bool LOAD = decltype(loads)::value;
    const int past = LOAD ? ends.past(uniform(stage)) : 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[u][i], x[u][j], acc[j][i], 0, 0, 0);
        if (LOAD && i & 1) {
          pin();
          load(dst, stage, from + 2 * j + i / 2, past);
          pin();
        }
      }
    pin();
  };
  auto multiply = [&](int u) { products(std::false_type(), u, nullptr, 0, 0); };
  auto multiply_and_load = [&](int u, int8_t* dst, int stage, int from) { products(std::true_type(), u, dst, stage, from); };
  // A stage in `cur`, its first operands on their way to w[0], x[0], half of the next in `next` and the other
  // half asked for here.  Before the barrier everyone's part of `next` is there and nobody reads `cur` any
  // more, of which `after` then fills half.
  auto step = [&](auto last, int8_t* cur, int8_t* next, int stage, int after) {
    constexpr bool LAST = decltype(last)::value;
    fetch(cur, 1);
    pin();
    multiply_and_load(0, next, stage, 4);
    fetch(cur, 2);
    pin();
    multiply(1);
    fetch(cur, 3);
    pin();
    multiply(0);
    wait_loads<0>();
    barrier();
    pin();
    if (!LAST) fetch(next, 0);
    pin();
    if (QKV && LAST) multiply(1);  // (the epilogue uses `cur`)
    else multiply_and_load(1, cur, after, 0);
  };
  Tile t = tile_at<WIDE, WIDE, WIDE_BAND>(a, first + slot);
  aim(t);
#pragma unroll
  for (int j = 0; j < WIDE_LOADS; ++j) load(lds0, 0, j, ends.past(0));
#pragma unroll
  for (int j = 0; j < WIDE_LOADS / 2; ++j) load(lds1, 1, j, ends.past(1));
  wait_loads<WIDE_LOADS / 2>();
  barrier();
  for (int parity = 0;; parity ^= 1) {
    const Tile done = t;
    const Set& s = a.set[done.set];
    load_channels<F16, QKV>(a, s, done.c0, channel[parity]);  // (read after the next barriers)
    float scale[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) scale[j] = s.scale[min(done.t0 + wt * 64 + j * 32 + col, s.tokens - 1)];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = i32x16{};
    fetch(lds0, 0);
    for (int n = 2; n < stages; n += 2) {
      step(std::false_type(), lds0, lds1, n - 1, n);
      step(std::false_type(), lds1, lds0, n, n + 1);
    }
    slot += stride;
    const bool more = slot < a.tiles_xcd && first + slot < a.tiles;
    // (the second half of this tile's last stage goes by its own addresses)
    fetch(lds0, 1);
    pin();
    multiply_and_load(0, lds1, stages - 1, 4);
    if (more) t = tile_at<WIDE, WIDE, WIDE_BAND>(a, first + slot);
    aim(t);  // (after the last tile: its own first stages once more, never read)
    fetch(lds0, 2);
    pin();
    multiply(1);
    fetch(lds0, 3);
    pin();
    multiply(0);
    wait_loads<0>();
    barrier();
    pin();
    fetch(lds1, 0);
    pin();
    multiply_and_load(1, lds0, 0, 0);
    step(std::true_type(), lds1, lds0, 0, 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float* const values = &channel[parity][0][wc * 128];
      const int c0 = done.c0 + wc * 128;
      const uint32_t t0 = done.t0 + wt * 64 + j * 32;
      if (!QKV) finish<F16, GELU, 4, WIDE>(a, s, acc[j], scale[j], values, c0, t0);
      else if (c0 < a.columns && a.cos && c0 < 2 * a.heads * HEAD) finish_head<F16, true, WIDE>(a, s, acc[j], scale[j], values, c0, t0, lds1 + 1024 * wave);
      else if (c0 < a.columns) finish_head<F16, false, WIDE>(a, s, acc[j], scale[j], values, c0, t0, lds1 + 1024 * wave);
    }
    if (QKV) {
#pragma unroll
      for (int j = 0; j < WIDE_LOADS / 2; ++j) load(lds1, 1, j, ends.past(1));
    }
    if (!more) break;
  }
  wait_loads<0>();  // (nothing may still be on its way to LDS when the workgroup ends)
}

// ------------------------------------------------------------------ fewer rows
// TC channels x TT tokens a workgroup, in tiles so small that most CUs have one.  What is on its way to a CU
// bounds it: some 70 to 100 bytes a ns and CU with 60 to 140 KB asked for ahead.  So the operands go to LDS by
// direct loads, into a ring of R stages of 128 features, as many as there is room for (straight into registers,
// which hold less: 1 x 3072 x 9216 qkv 15.3 us, so 10.9; 77 x 4096 x 3072 12.4 -> 9.6), the loads spread over the
// products.  A stage's features are in four parts of 32, a wave each in the smallest tiles (77 x 4096 x 3072 10.3 us
// with two), or two waves that share the tokens (of 32 tokens: the channels), whose epilogue is shorter
// (512 x 3072 x 9216 28.8 us, with one 33.6).  The sums meet in LDS, and a thread finishes eight channels of a
// token: neighbouring lanes read and write whole lines (a wave finishing 32 tokens as they lie in registers:
// 512 + 1024 x 3072 qkv 88 us of 128 x 128 tiles, so 73).  Rows past the operands' ends are zeros that nothing reads.
template <int TC, int TT, int WAVES>
struct Ring {
  static constexpr int STAGE = (TC + TT) * 128, GROUPS = STAGE / 1024, LOADS = (GROUPS + WAVES - 1) / WAVES;
  static constexpr int CW = TT > 32 ? TC : TC / 2, TW = TT > 32 ? TT / 2 : TT;  // of half the sums
  static constexpr int BOX = TW * CW * 4;
  static constexpr int CF = (WAVES > 4 ? CW : TC) / 32, TF = (WAVES > 4 ? TW : TT) / 32;  // of a wave
};

template <bool F16, bool QKV, bool GELU, int TC, int TT, int R, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void int8_tile_kernel(Args a) {
  typedef Ring<TC, TT, WAVES> F;
  constexpr int STAGE = F::STAGE, LOADS = F::LOADS, CW = F::CW, TW = F::TW, CF = F::CF, TF = F::TF;
  static_assert(F::BOX <= STAGE && R >= 4 && R <= 8, "a stage holds half a part's sums");
  __shared__ __attribute__((aligned(1024))) int8_t lds0[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds1[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds2[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds3[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds4[R > 4 ? STAGE : 1];
  __shared__ __attribute__((aligned(1024))) int8_t lds5[R > 5 ? STAGE : 1];
  __shared__ __attribute__((aligned(1024))) int8_t lds6[R > 6 ? STAGE : 1];
  __shared__ __attribute__((aligned(1024))) int8_t lds7[R > 7 ? STAGE : 1];
  __shared__ __attribute__((aligned(16))) float channel[3][TC];
  auto ring = [&](auto index) -> int8_t* {
    constexpr int i = decltype(index)::value % R;
    return i == 0 ? lds0 : i == 1 ? lds1 : i == 2 ? lds2 : i == 3 ? lds3 : i == 4 ? lds4 : i == 5 ? lds5 : i == 6 ? lds6 : lds7;
  };
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int part = WAVES > 4 ? wave >> 1 : wave, share = WAVES > 4 ? wave & 1 : 0;
  const uint32_t tile = (blockIdx.x & 7) * a.tiles_xcd + (blockIdx.x >> 3);
  if (tile >= a.tiles) return;
  const Tile t = tile_at<TC, TT, 8>(a, tile);
  const Set& s = a.set[t.set];
  load_channels<F16, QKV>(a, s, t.c0, channel);
  // Loads as in the wide kernel.
  const int8_t *wbase = s.w + (int64_t)t.c0 * a.padded, *qbase = s.q + (int64_t)t.t0 * a.padded;
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  int offset[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = 8 * (WAVES * j + wave) + (lane >> 3);
    const bool there = r < TC ? r < a.columns - t.c0 : (uint32_t)(r - TC) < s.tokens - t.t0;
    offset[j] = there ? (r < TC ? r : r - TC) * a.padded + chunk * 16 : (int)0x80000000;
  }
  const int stages = (a.padded + 127) / 128;
  const Ends ends(a.padded, chunk);
  const bool all = WAVES * (LOADS - 1) + wave < F::GROUPS;  // (the last loads are not every wave's)
  auto load = [&](int8_t* dst, int stage, int j, int past) {
    const int group = WAVES * j + wave;
    if (F::GROUPS % WAVES == 0 || j < LOADS - 1 || all)
      load_lds16(group * 8 < TC ? wbase : qbase, dst + 1024 * group, offset[j] | past, uniform(stage * 128));
  };
  auto arrivals = [&] {
    if (F::GROUPS % WAVES == 0 || all) wait_arrivals<(R - 3) * LOADS>();
    else wait_arrivals<(R - 3) * (LOADS - 1)>();
  };
  const int read = col * 128 + ((col >> 1 & 7) ^ (2 * part + half)) * 16;
  const int wread = read + (TT > 32 ? 0 : share * CW * 128), xread = read + (TC + (TT > 32 ? share * TW : 0)) * 128;
  i32x4 w[2][CF], x[2][TF];
  auto fetch = [&](const int8_t* src, int to) {
#pragma unroll
    for (int i = 0; i < CF; ++i) w[to][i] = *(const i32x4*)(src + wread + i * 4096);
#pragma unroll
    for (int j = 0; j < TF; ++j) x[to][j] = *(const i32x4*)(src + xread + j * 4096);
    __builtin_amdgcn_sched_barrier(0);
  };
  i32x16 acc[TF][CF] = {};
  // Stage n's operands are in w, x, or on their way; stage n + 1 is in LDS.  The stage whose reads ended in
  // the last step takes n + R - 1.  Before the barrier stage n + 2 is there.
  int n = 0;
  auto step = [&](auto index) {
    constexpr int I = decltype(index)::value;
    int8_t* const free = ring(std::integral_constant<int, I + R - 1>());
    const int past = ends.past(uniform(n + R - 1));
    int asked = 0, done = 0;
#pragma unroll
    for (int j = 0; j < TF; ++j)
#pragma unroll
      for (int i = 0; i < CF; ++i) {
        acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[I & 1][i], x[I & 1][j], acc[j][i], 0, 0, 0);
        for (++done; asked * TF * CF < done * LOADS; ++asked) {
          __builtin_amdgcn_sched_barrier(0);
          load(free, n + R - 1, asked, past);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    fetch(ring(std::integral_constant<int, I + 1>()), ~I & 1);
    arrivals();
    barrier();
    return ++n == stages;
  };
  // (Zeros into the last stage, so that the compiler, which tracks what is on its way to which array, has met them
  // all before the loop: otherwise it waits for everything each time around.)
  load(ring(std::integral_constant<int, R - 1>()), 0, 0, (int)0x80000000);
  auto begin = [&](auto index) {
    constexpr int I = decltype(index)::value;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load(ring(index), I, j, ends.past(I));
  };
  begin_all(begin, std::make_integer_sequence<int, R - 1>());
  arrivals();
  barrier();
  fetch(lds0, 0);
  while (!step_all(step, std::make_integer_sequence<int, R % 2 ? 2 * R : R>())) {}
  wait_loads<0>();  // (nothing is on its way to LDS any more)
  barrier();
  // Parts 2 and 3 hand their sums to 0 and 1, which add their own: token-major, four channels a unit, units in an
  // order of the token's, so that neighbouring tokens' lie in different banks.
  auto box = [&](int k, int h) -> int8_t* { return k ? (h ? lds3 : lds2) : (h ? lds1 : lds0); };
  auto unit = [&](int token, int c) { return (token * CW + (c ^ (token & 7) * 4)) * 4; };
  auto hand = [&](bool add) {
#pragma unroll
    for (int j = 0; j < TF; ++j)
#pragma unroll
      for (int i = 0; i < CF; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int h = WAVES > 4 ? share : TT > 32 ? j * 32 / TW : i * 32 / CW;
          const int token = TT > 32 ? j * 32 % TW : j * 32, c = TT > 32 ? i * 32 : i * 32 % CW;
          i32x4* const at = (i32x4*)(box(part & 1, h) + unit(token + col, c + g * 8 + half * 4));
          const i32x4 v = {acc[j][i][4 * g], acc[j][i][4 * g + 1], acc[j][i][4 * g + 2], acc[j][i][4 * g + 3]};
          *at = add ? *at + v : v;
        }
  };
  if (part >= 2) hand(false);
  __syncthreads();
  if (part < 2) hand(true);
  __syncthreads();
  for (int e = threadIdx.x; e < TT * (TC / 8); e += 64 * WAVES) {
    const int token = e / (TC / 8), c = e % (TC / 8) * 8;
    const int h = TT > 32 ? token / TW : c / CW;
    i32x4 sum[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int at = unit(TT > 32 ? token % TW : token, (TT > 32 ? c : c % CW) + 4 * g);
      sum[g] = *(const i32x4*)(box(0, h) + at) + *(const i32x4*)(box(1, h) + at);
    }
    const uint32_t to = t.t0 + token;
    finish8<F16, QKV, GELU, TC>(a, s, sum, s.scale[min(to, s.tokens - 1)], channel, t.c0, to, c);
  }
}

// ------------------------------------------------------------------ a few rows of 16 bits
// Linear layer of rows that are quantized here, by every workgroup for itself: few enough that this hides behind
// the first weights' way to it, and saves a launch.  TC channels a workgroup of four waves, a part of a stage's
// features each; a ring of R stages of the weight alone, three workgroups a CU.  Bound by the weight's read: 1 x 3072 x
// 18432 (57 MB) 11.5 us, 4.9 TB/s (64 channels, six stages: 12.3; 32768 values of rows in LDS, two workgroups a CU:
// 17.1); small ones by the launch, 1 x 512 x 2048 6.0.
constexpr int FEW_ROWS = 32, FEW_VALUES = HB_INT8_FEW_VALUES;

struct FewArgs {
  Args a;  // (its one set has neither q nor scale)
  const uint16_t* x;
  int64_t x_b, x_n;
  int32_t features;
};

template <bool F16, bool GELU, int TC, int R>
__global__ __launch_bounds__(256, 2) void int8_few_kernel(FewArgs f) {
  constexpr int STAGE = TC * 128, LOADS = STAGE / 4096, CF = TC / 32, VECTORS = FEW_VALUES / 2048;
  static_assert(R == 6 || R == 8, "an even ring");
  __shared__ __attribute__((aligned(1024))) int8_t lds0[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds1[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds2[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds3[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds4[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds5[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds6[R > 6 ? STAGE : 1];
  __shared__ __attribute__((aligned(1024))) int8_t lds7[R > 7 ? STAGE : 1];
  __shared__ __attribute__((aligned(16))) int8_t rows[FEW_VALUES];
  __shared__ __attribute__((aligned(16))) float channel[3][TC];
  __shared__ uint32_t groups[FEW_VALUES / 64], tops[FEW_ROWS];
  __shared__ float scales[FEW_ROWS];
  auto ring = [&](auto index) -> int8_t* {
    constexpr int i = decltype(index)::value % R;
    return i == 0 ? lds0 : i == 1 ? lds1 : i == 2 ? lds2 : i == 3 ? lds3 : i == 4 ? lds4 : i == 5 ? lds5 : i == 6 ? lds6 : lds7;
  };
  const Args& a = f.a;
  const Set& s = a.set[0];
  const int lane = threadIdx.x & 63, part = uniform(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int c0 = blockIdx.x * TC;
  // The rows' values, asked for before any weights: eight at a time, a row's after the one's before it.
  const int padded = a.padded, row_bytes = (padded + 127) & ~127;  // (in LDS)
  const uint32_t each = (uint32_t)padded / 8, all = s.tokens * each;
  auto row_at = [&](uint32_t r) {
    const uint32_t b = r / s.rows;
    return f.x + b * f.x_b + (int64_t)(r - b * s.rows) * f.x_n;
  };
  u32x4 raw[VECTORS];
  uint32_t row[VECTORS];
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    const uint32_t at = v * 256 + threadIdx.x;
    row[v] = at / each;
    raw[v] = u32x4{0, 0, 0, 0};
    const int c = (int)(at - row[v] * each) * 8;
    if (at < all) raw[v] = *(const any_u32x4*)(row_at(row[v]) + min(c, f.features - 8));
  }
  // (load_channels, whose loads have to be asked for before those to LDS too)
  const int mine = min(c0 + (int)threadIdx.x % TC, a.columns - 1);
  const float weight_scale = s.w_scale[mine];
  const uint16_t bias = (s.bias ? s.bias : (const uint16_t*)s.w_scale)[mine];  // (a value unused; no branch to wait at)
  // Loads of the weight as in the tile kernel.
  const int8_t* const wbase = s.w + (int64_t)c0 * padded;
  const int chunk = (lane & 7) ^ ((4 * part + (lane >> 4)) & 7);
  int offset[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = 8 * (4 * j + part) + (lane >> 3);
    offset[j] = r < a.columns - c0 ? r * padded + chunk * 16 : (int)0x80000000;
  }
  const int stages = (padded + 127) / 128;
  const Ends ends(padded, chunk);
  auto load = [&](int8_t* dst, int stage, int j, int past) {
    load_lds16(wbase, dst + 1024 * (4 * j + part), offset[j] | past, uniform(stage * 128));
  };
  // (Zeros into the last stage as above.)
  load(ring(std::integral_constant<int, R - 1>()), 0, 0, (int)0x80000000);
  auto begin = [&](auto index) {
    constexpr int I = decltype(index)::value;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load(ring(index), I, j, ends.past(I));
  };
  begin_all(begin, std::make_integer_sequence<int, R - 1>());
  // The rows' largest patterns: of eight lanes, which are always of one row, then of a row's groups of those.
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    const int c = (int)(v * 256 + threadIdx.x - row[v] * each) * 8, past = c + 8 - f.features;
    if (past > 0) raw[v] = drop_values(raw[v], min(past, 8));  // (what lies before a row's last values)
    uint32_t top = fp32_bits<F16>(max_pairs(u16x2{0, 0}, raw[v]));
    top = max(top, moved_bits<0xb1>(top));
    top = max(top, moved_bits<0x4e>(top));
    top = max(top, moved_bits<0x141>(top));
    if ((lane & 7) == 0) groups[v * 32 + (threadIdx.x >> 3)] = top;
  }
  if (threadIdx.x < TC) {
    channel[0][threadIdx.x] = weight_scale;
    channel[1][threadIdx.x] = s.bias ? to_f<F16>(bias) : 0.f;
  }
  wait_loads<63>();
  barrier();
  for (uint32_t m = part; m < s.tokens; m += 4) {
    uint32_t top = 0;
    for (uint32_t k = lane; k < each / 8; k += 64) top = max(top, groups[m * (each / 8) + k]);
    top = max(top, moved_bits<0xb1>(top));
    top = max(top, moved_bits<0x4e>(top));
    top = max(top, moved_bits<0x141>(top));
    top = max(top, moved_bits<0x140>(top));
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    if (lane == 0) tops[m] = top;
  }
  wait_loads<63>();
  barrier();
  // Their whole numbers: chunks of 16 bytes, each 128 bytes' in an order of the row's, so that rows lie in
  // different banks.
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    const uint32_t at = v * 256 + threadIdx.x;
    if (at < all) {
      const Scaler scaler(tops[row[v]]);
      const int c = (int)(at - row[v] * each) * 8;
      float values[8];
      unpack8<F16>(raw[v], values);
      *(u32x2*)(rows + row[v] * row_bytes + (c & ~127) + ((c >> 4 & 7) ^ (row[v] & 7)) * 16 + (c & 8)) = pack_row8(scaler, values);
      if (c == 0) scales[row[v]] = scaler.scale;
    }
  }
  wait_loads<63>();
  wait_arrivals<(R - 3) * LOADS>();
  barrier();
  const int read = col * 128 + ((col >> 1 & 7) ^ (2 * part + half)) * 16;
  const int token = min(col, (int)s.tokens - 1), xread = token * row_bytes + ((2 * part + half) ^ (token & 7)) * 16;
  i32x4 w[2][CF], x[2];
  auto fetch = [&](const int8_t* src, int stage, int to) {
#pragma unroll
    for (int i = 0; i < CF; ++i) w[to][i] = *(const i32x4*)(src + read + i * 4096);
    x[to] = *(const i32x4*)(rows + xread + min(stage, stages - 1) * 128);
    __builtin_amdgcn_sched_barrier(0);
  };
  i32x16 acc[CF] = {};
  int n = 0;
  auto step = [&](auto index) {
    constexpr int I = decltype(index)::value;
    int8_t* const free = ring(std::integral_constant<int, I + R - 1>());
    const int past = ends.past(uniform(n + R - 1));
#pragma unroll
    for (int i = 0; i < CF; ++i) {
      acc[i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[I & 1][i], x[I & 1], acc[i], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      load(free, n + R - 1, i, past);
      __builtin_amdgcn_sched_barrier(0);
    }
    fetch(ring(std::integral_constant<int, I + 1>()), n + 1, ~I & 1);
    wait_arrivals<(R - 3) * LOADS>();
    barrier();
    return ++n == stages;
  };
  static_assert(LOADS == CF, "a load a product");
  fetch(lds0, 0, 0);
  while (!step_all(step, std::make_integer_sequence<int, R>())) {}
  wait_loads<0>();  // (nothing is on its way to LDS any more)
  barrier();
  // The four parts' sums, [token][channel], each in a stage.
  int8_t* const box = part == 0 ? lds0 : part == 1 ? lds1 : part == 2 ? lds2 : lds3;
  if (col < (int)s.tokens) {
#pragma unroll
    for (int i = 0; i < CF; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(i32x4*)(box + (col * TC + ((i * 32 + g * 8 + half * 4) ^ (col & 7) * 4)) * 4) =
            i32x4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < s.tokens * (TC / 8); e += 256) {
    const uint32_t to = e / (TC / 8);
    const int c = e % (TC / 8) * 8;
    i32x4 sum[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int at = (to * TC + ((c + 4 * g) ^ (to & 7) * 4)) * 4;
      sum[g] = *(const i32x4*)(lds0 + at) + *(const i32x4*)(lds1 + at) + *(const i32x4*)(lds2 + at) + *(const i32x4*)(lds3 + at);
    }
    finish8<F16, false, GELU, TC>(a, s, sum, scales[to], channel, c0, to, c);
  }
}

// ------------------------------------------------------------------ launches
enum Kernel { T64x32, T32x64, T64x64, T96x64, T96x128, T128x32, T128x64, T128x128, WIDE256, WIDE_HEADS, KERNELS };

// What a tile of each kernel covers, and what it takes on 256 CUs, a whole MI355X (on a partition of one the results are
// the same, the choice untimed), fitted to the times of 694 linear and 30 Q/K/V sizes of 1 to 6000 rows: `launch`,
// and for a round of tiles, one a CU, `round` + stages of 128 features x (`stage` + `full` f^2) us, f the share of the
// CUs that have one (stages slow each other down where many load).
struct Shape {
  int tc, tt;
  float launch, round, stage, full;
};
constexpr Shape SHAPES[KERNELS] = {
    // linear
    {64, 32, 2.97f, 1.34f, 0.102f, 0.065f},
    {32, 64, 1.81f, 2.61f, 0.096f, 0.088f},
    {64, 64, 1.74f, 2.84f, 0.127f, 0.134f},
    {96, 64, 1.67f, 3.78f, 0.189f, 0.133f},
    {96, 128, 0.95f, 5.82f, 0.258f, 0.234f},
    // qkv (a head's channels stay together)
    {128, 32, 1.91f, 3.63f, 0.174f, 0.138f},
    {128, 64, 1.96f, 4.70f, 0.195f, 0.249f},
    {128, 128, 1.91f, 6.67f, 0.304f, 0.349f},
    // the wide kernel, linear and qkv
    {256, 256, 5.9f, 3.0f, 0.99f, 0.70f},
    {256, 256, 7.0f, 8.2f, 1.00f, 0.70f},
};

// Tiles of TC x TT of both sets.
int64_t tiles_of(const Args& a, int count, int tc, int tt) {
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i)
    tiles += ((a.set[i].tokens + (int64_t)tt - 1) / tt) * ((a.columns + (int64_t)tc - 1) / tc);
  return tiles;
}

// What a kernel takes for the sets, in us.
float estimate(const Args& a, int count, Kernel k) {
  const Shape& s = SHAPES[k];
  const float rounds = (float)tiles_of(a, count, s.tc, s.tt) / 256.f, whole = std::floor(rounds), rest = rounds - whole;
  const float stages = (float)((a.padded + 127) / 128);
  return s.launch + whole * (s.round + stages * (s.stage + s.full)) +
         (rest > 0.f ? s.round + stages * (s.stage + s.full * rest * rest) : 0.f);
}

struct Choice {
  Kernel kernel;
  float us;
};

// The kernel whose estimate is the least: over the linear sizes 0.5% slower than always the fastest, at worst 21%
// (30 x 8760 x 4433); for all 30 Q/K/V sizes it is the fastest, few as they are.  Measured, rows x features x
// columns, us for 64 x 32 / 32 x 64 / 64 x 64 / 96 x 64 / 96 x 128 / 256 x 256 tiles: 77 x 4096 x 3072 9.5 / 9.0 /
// 10.1 / 12.2 / 15.3 / 40; 128 x 3072 x 12288 18 / 21 / 17 / 12.1 / 15.5 / 32; 512 x 12288 x 3072 45 / 54 / 45 /
// 28.8 / 37 / 108; 666 x 1000 x 777 6.9 / 8.9 / 6.4 / 7.4 / 9.6 / 18; 256 x 3072 x 9216 25 / 32 / 23 / 20 / 15.4 /
// 33; 4096 x 3072 x 3072 96 / 141 / 86 / 74 / 56 / 38; 1 x 3072 x 18432 13.4 / 19.5 / 17.0 / 12.8 / 14.1 / 31.
// qkv, rows x features, 24 heads, us for 128 x 32 / 128 x 64 / 128 x 128 / 256 x 256: 1 x 3072 11.2 / 12.0 / 15.9 /
// 37; 128 x 3072 21 / 14.7 / 19.3 / 41; 512 x 3072 48 / 37 / 36 / 43; 512 + 4096 x 3072 365 / 236 / 192 / 141.
Choice choose(const Args& a, int count, bool qkv) {
  const Kernel wide = qkv ? WIDE_HEADS : WIDE256;
  Choice best = {wide, estimate(a, count, wide)};
  for (int i = qkv ? T128x32 : T64x32; i <= (qkv ? T128x128 : T96x128); ++i) {
    const Kernel k = (Kernel)i;
    if (tiles_of(a, count, SHAPES[k].tc, SHAPES[k].tt) >= (1 << 21)) continue;  // (a grid holds fewer than 2^32 threads)
    const float us = estimate(a, count, k);
    if (us < best.us) best = {k, us};
  }
  return best;
}

// The last rows of the last set that are better off in a launch of their own, because the tiles before them
// fill whole rounds of the CUs: 16896 x 15360 x 3072, 792 tiles of 256 x 256, 788 us at once, and 675 as
// 768 of them and 512 rows apart.
uint32_t apart(const Args& a, int count, const Choice& whole, bool qkv) {
  const Set& s = a.set[count - 1];
  const int64_t across = (a.columns + 255) / 256, tiles = tiles_of(a, count, 256, 256);
  if (whole.kernel < WIDE256 || tiles < 256 || tiles % 256 == 0) return 0;
  // token tiles to take off, so that what is left is the most that fits the whole rounds
  const int64_t off = (tiles % 256 + across - 1) / across, token_tiles = (s.tokens + 255) / 256;
  if (off >= token_tiles) return 0;
  const uint32_t keep = (uint32_t)(token_tiles - off) * 256;
  Args main = a, rest = a;
  main.set[count - 1].tokens = keep;
  rest.set[0] = s;
  rest.set[0].tokens = s.tokens - keep;
  return estimate(main, count, whole.kernel) + choose(rest, 1, qkv).us + 5.f < whole.us ? s.tokens - keep : 0;
}

template <bool F16, bool QKV, bool GELU>
int launch_kernel(Args& a, int count, Kernel kernel, hipStream_t st) {
  const int tc = SHAPES[kernel].tc, tt = SHAPES[kernel].tt;
  const int64_t tiles = tiles_of(a, count, tc, tt);
  HB_REQUIRE(tiles < (1ll << 30), "too many output tiles for one launch");
  a.channel_tiles = (uint32_t)((a.columns + tc - 1) / tc);
  a.tiles0 = (uint32_t)tiles_of(a, 1, tc, tt);
  a.tiles = (uint32_t)tiles;
  a.tiles_xcd = (a.tiles + 7) / 8;
  const dim3 each(8 * a.tiles_xcd), four(256), eight(512);
  switch (kernel) {
    case T64x32:
      if constexpr (!QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 64, 32, 6, 4>), each, four, 0, st, a);
      break;
    case T32x64:
      if constexpr (!QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 32, 64, 8, 4>), each, four, 0, st, a);
      break;
    case T64x64:
      if constexpr (!QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 64, 64, 8, 8>), each, eight, 0, st, a);
      break;
    case T96x64:
      if constexpr (!QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 96, 64, 7, 8>), each, eight, 0, st, a);
      break;
    case T96x128:
      if constexpr (!QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 96, 128, 5, 8>), each, eight, 0, st, a);
      break;
    case T128x32:
      if constexpr (QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 128, 32, 7, 8>), each, eight, 0, st, a);
      break;
    case T128x64:
      if constexpr (QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 128, 64, 6, 8>), each, eight, 0, st, a);
      break;
    case T128x128:
      if constexpr (QKV) hipLaunchKernelGGL((int8_tile_kernel<F16, QKV, GELU, 128, 128, 4, 8>), each, eight, 0, st, a);
      break;
    default: {
      const uint32_t per_xcd = std::max(1, device_cu_count() / 8);
      hipLaunchKernelGGL((int8_wide_kernel<F16, QKV, GELU>), dim3(8 * std::min(a.tiles_xcd, per_xcd)), eight, 0, st, a);
    }
  }
  HB_HIP(hipGetLastError());
  return HB_OK;
}

template <bool F16, bool QKV, bool GELU>
int launch_type(Args& a, int count, hipStream_t st) {
  const Choice whole = choose(a, count, QKV);
  const uint32_t rest = apart(a, count, whole, QKV);
  if (!rest) return launch_kernel<F16, QKV, GELU>(a, count, whole.kernel, st);
  Args b = a;
  Set& s = b.set[0] = a.set[count - 1];
  a.set[count - 1].tokens -= rest;
  s.start = s.tokens - rest;
  s.q += (int64_t)s.start * a.padded;
  s.scale += s.start;
  s.tokens = rest;
  const int rc = launch_kernel<F16, QKV, GELU>(a, count, whole.kernel, st);
  return rc ? rc : launch_kernel<F16, QKV, GELU>(b, 1, choose(b, 1, QKV).kernel, st);
}

template <bool QKV>
int launch(Args& a, int count, int32_t dtype, hipStream_t st) {
  if constexpr (QKV)
    return dtype == HB_DTYPE_F16 ? launch_type<true, true, false>(a, count, st) : launch_type<false, true, false>(a, count, st);
  else if (dtype == HB_DTYPE_F16)
    return a.gelu ? launch_type<true, false, true>(a, count, st) : launch_type<true, false, false>(a, count, st);
  else
    return a.gelu ? launch_type<false, false, true>(a, count, st) : launch_type<false, false, false>(a, count, st);
}

template <bool F16, bool GELU>
int launch_few(const FewArgs& f, hipStream_t st) {
  hipLaunchKernelGGL((int8_few_kernel<F16, GELU, 32, 8>), dim3((f.a.columns + 31) / 32), dim3(256), 0, st, f);
  HB_HIP(hipGetLastError());
  return HB_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The checks both entry points make of a set's rows and weight.
int check_set(const Set& s, int32_t batch, int32_t rows, int32_t padded) {
  HB_REQUIRE(batch > 0 && rows > 0 && (int64_t)batch * rows < (1ll << 31), "batch and rows must be positive, with fewer than 2^31 rows in all");
  HB_REQUIRE(s.q && s.scale && s.w && s.w_scale && s.out, "null pointer argument");
  HB_REQUIRE(aligned16(s.q) && aligned16(s.w), "rows and weights must be 16-byte aligned");
  HB_REQUIRE(((uintptr_t)s.scale & 3) == 0 && ((uintptr_t)s.w_scale & 3) == 0, "scales must be 4-byte aligned");
  HB_REQUIRE(((uintptr_t)s.bias & 1) == 0 && ((uintptr_t)s.out & 1) == 0, "bias and output must be 2-byte aligned");
  HB_REQUIRE(padded > 0 && padded % 64 == 0 && padded <= MAX_FEATURES, "padded must be a positive multiple of 64 up to %d (got %d)", MAX_FEATURES, padded);
  HB_REQUIRE(s.out_b >= 0 && s.out_n >= 0, "output strides must be non-negative");
  return HB_OK;
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int hb_int8_linear(int32_t count, int32_t batch, const int32_t* rows, int32_t columns, int32_t padded,
                              int32_t dtype, int32_t gelu, void* const* pointers, const int64_t* strides,
                              hb_stream_t stream) {
  HB_REQUIRE(count == 1 || count == 2, "count must be 1 or 2");
  HB_REQUIRE(rows && pointers && strides, "null pointer argument");
  HB_REQUIRE(columns > 0 && columns < (1 << 30), "columns must be positive (and below 2^30)");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16, "dtype must be bf16 or fp16");
  HB_REQUIRE(gelu == 0 || gelu == 1, "gelu must be 0 or 1");
  Args a = {};
  a.columns = columns;
  a.padded = padded;
  a.gelu = gelu;
  a.vectors = 1;
  for (int i = 0; i < count; ++i) {
    void* const* p = pointers + 6 * i;
    Set& s = a.set[i];
    s = {(const int8_t*)p[0], (const float*)p[1], (const int8_t*)p[2], (const float*)p[3], (const uint16_t*)p[4],
         (uint16_t*)p[5], {nullptr, nullptr}, strides[2 * i], strides[2 * i + 1], (uint32_t)rows[i], 0, 0, 0};
    const int rc = check_set(s, batch, rows[i], padded);
    if (rc) return rc;
    s.tokens = (uint32_t)(batch * rows[i]);
    a.vectors &= aligned16(s.out) && s.out_b % 8 == 0 && s.out_n % 8 == 0;
  }
  return launch<false>(a, count, dtype, stream);
}

extern "C" int hb_int8_linear_rows(const void* x, int64_t batch_stride, int64_t row_stride, int32_t batch, int32_t rows,
                                   int32_t features, int32_t columns, int32_t padded, int32_t dtype, int32_t gelu,
                                   const int8_t* weight, const float* weight_scale, const void* bias, void* out,
                                   int64_t out_batch_stride, int64_t out_row_stride, hb_stream_t stream) {
  HB_REQUIRE(x && weight && weight_scale && out, "null pointer argument");
  HB_REQUIRE(batch > 0 && rows > 0 && batch <= FEW_ROWS && rows <= FEW_ROWS && batch * rows <= FEW_ROWS, "batch and rows must be positive, with at most %d rows in all", FEW_ROWS);
  HB_REQUIRE(features >= 8, "at least 8 features");
  HB_REQUIRE(padded >= features && padded % 64 == 0 && padded <= FEW_VALUES, "padded must be a multiple of 64, no smaller than features");
  HB_REQUIRE(batch * rows * ((padded + 127) / 128 * 128) <= FEW_VALUES, "at most %d values of rows in all", FEW_VALUES);
  HB_REQUIRE(columns > 0 && columns < (1 << 28), "columns must be positive (and below 2^28)");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16, "dtype must be bf16 or fp16");
  HB_REQUIRE(gelu == 0 || gelu == 1, "gelu must be 0 or 1");
  HB_REQUIRE((((uintptr_t)x | (uintptr_t)bias | (uintptr_t)out) & 1) == 0 && aligned16(weight) && ((uintptr_t)weight_scale & 3) == 0,
             "x, bias and out must be 2-byte, the weight 16-byte and its scales 4-byte aligned");
  HB_REQUIRE(batch_stride >= 0 && row_stride >= 0 && out_batch_stride >= 0 && out_row_stride >= 0, "strides must be non-negative");
  FewArgs f = {};
  f.x = (const uint16_t*)x;
  f.x_b = batch_stride;
  f.x_n = row_stride;
  f.features = features;
  Args& a = f.a;
  a.columns = columns;
  a.padded = padded;
  a.gelu = gelu;
  a.vectors = aligned16(out) && out_batch_stride % 8 == 0 && out_row_stride % 8 == 0;
  a.set[0] = {nullptr, nullptr, weight, weight_scale, (const uint16_t*)bias, (uint16_t*)out, {nullptr, nullptr},
              out_batch_stride, out_row_stride, (uint32_t)rows, (uint32_t)(batch * rows), 0, 0};
  if (dtype == HB_DTYPE_F16) return gelu ? launch_few<true, true>(f, stream) : launch_few<true, false>(f, stream);
  return gelu ? launch_few<false, true>(f, stream) : launch_few<false, false>(f, stream);
}

extern "C" int hb_int8_qkv(int32_t batch, int32_t text_tokens, int32_t tokens, int32_t heads, int32_t padded,
                           int32_t dtype, float eps, void* const* pointers, const float* cos, const float* sin,
                           void* out, int64_t out_plane_stride, int64_t out_batch_stride, int64_t out_row_stride,
                           hb_stream_t stream) {
  HB_REQUIRE(pointers && out, "null pointer argument");
  HB_REQUIRE(tokens > 0 && text_tokens >= 0 && text_tokens < tokens, "tokens must be positive with 0 <= text_tokens < tokens");
  HB_REQUIRE(heads > 0 && heads <= (1 << 20), "heads must be in [1, 2^20]");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16, "dtype must be bf16 or fp16");
  HB_REQUIRE(eps > 0.f, "eps must be positive");
  HB_REQUIRE((cos == nullptr) == (sin == nullptr), "cos and sin must be given together");
  HB_REQUIRE(aligned16(out) && aligned16(cos) && aligned16(sin), "out, cos and sin must be 16-byte aligned");
  const int64_t strides[3] = {out_plane_stride, out_batch_stride, out_row_stride};
  for (int i = 0; i < 3; ++i)
    HB_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "output strides must be non-negative multiples of 8");
  Args a = {};
  a.columns = 3 * heads * HEAD;
  a.padded = padded;
  a.vectors = 1;
  a.cos = cos;
  a.sin = sin;
  a.out_p = out_plane_stride;
  a.heads = heads;
  a.eps = eps;
  int count = 0;
  for (int i = text_tokens == 0; i < 2; ++i) {
    void* const* p = pointers + 7 * i;
    const int32_t rows = i == 0 ? text_tokens : tokens - text_tokens, first = i == 0 ? 0 : text_tokens;
    Set& s = a.set[count++];
    s = {(const int8_t*)p[0], (const float*)p[1], (const int8_t*)p[2], (const float*)p[3], (const uint16_t*)p[4],
         (uint16_t*)out + first * out_row_stride, {(const uint16_t*)p[5], (const uint16_t*)p[6]}, out_batch_stride,
         out_row_stride, (uint32_t)rows, 0, (uint32_t)first, 0};
    const int rc = check_set(s, batch, rows, padded);
    if (rc) return rc;
    HB_REQUIRE(((uintptr_t)s.norm[0] & 1) == 0 && ((uintptr_t)s.norm[1] & 1) == 0, "norm weights must be 2-byte aligned");
    s.tokens = (uint32_t)(batch * rows);
  }
  return launch<true>(a, count, dtype, stream);
}
