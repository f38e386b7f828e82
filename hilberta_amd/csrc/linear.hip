// Linear layers of 16-bit rows with what follows them in the same pass.
//
//   out[m, n] = residual[m, n] + gate[b, n] * act(sum_k x[m, k] w[n, k] + bias[n])
//
// act: none, GELU(tanh) or SiLU; bias, residual and gate where they are given.  The sums are fp32 and so is what
// follows, rounded once to the 16-bit output.
//
// The weight's channels are the rows of the matrix instruction and the tokens its columns, as in the 8-bit products: a
// lane then holds one token's values, 4 consecutive channels an accumulator quarter.
//
// Three kernels: many rows (linear_wide_kernel), fewer (linear_tile_kernel) and a few (linear_few_kernel).  Where their
// tiles are few the first two take the features in parts, whose sums join_kernel adds; rows that direct loads cannot take
// are copied first (pad_rows_kernel).
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "gemm_common.h"
#include "rows16.h"
#include "../../include/hilberta_hip.h"

namespace hb {
namespace {

enum Act { NONE, GELU, SILU };

// One set of rows with its weight.  Two sets (a block's text and image rows) share a launch.
struct Set {
  const uint16_t* x;         // [tokens, features]
  const uint16_t* w;         // [columns, features]
  const uint16_t* bias;      // [columns] or null
  const uint16_t* residual;  // [tokens, columns] or null
  const uint16_t* gate;      // [batch, columns] or null
  uint16_t* out;
  int64_t x_b, x_n, w_n, r_b, r_n, g_b, out_b, out_n;  // strides of a batch element and a row
  uint32_t rows, tokens;     // rows of a batch element, and of all
};

struct Args {
  Set set[2];
  int32_t columns, features;
  uint32_t tiles0, tiles, tiles_xcd;  // tiles of set 0, of all, and of an XCD (in parts: of all parts)
  uint32_t channel_tiles;             // tiles along the channels
  int32_t act;
  int32_t vectors;                    // every output row takes 16-byte stores
  int32_t splits, stages_each;        // parts of the features, and stages of each
  float* sums;                        // [splits, tokens of both sets, columns rounded up to 8], with several parts
};

template <bool F16>
__device__ __forceinline__ f32x16 multiply32(const u32x4& w, const u32x4& x, const f32x16& acc) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f32x4 multiply16(const u32x4& w, const u32x4& x, const f32x4& acc) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
}

// The same with the sums in accumulation registers and the operands in the others: where 256 sums take all of the former,
// the compiler left to itself moves some to and fro in every stage (16384 x 12288 x 3072 846 -> 1070 us by a change in the
// order of loads).  It does not know these for matrix instructions and adds none of their waits, so whatever reads a sum
// next comes late enough by itself: the next product on it 64 products later, moved_out after settle.
template <bool F16>
__device__ __forceinline__ void accumulate16(const u32x4& w, const u32x4& x, f32x4& acc) {
  if constexpr (F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(w), "v"(x));
  else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(w), "v"(x));
}
template <bool F16>
__device__ __forceinline__ void begin16(const u32x4& w, const u32x4& x, f32x4& acc) {
  if constexpr (F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=a"(acc) : "v"(w), "v"(x));
  else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=a"(acc) : "v"(w), "v"(x));
}
// The last product's sums are there (18 cycles after a product of 8 passes).
__device__ __forceinline__ void settle() {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ float moved_out(float acc) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(acc));
  return v;
}
__device__ __forceinline__ f32x4 moved_out(const f32x4& acc) {
  return f32x4{moved_out(acc[0]), moved_out(acc[1]), moved_out(acc[2]), moved_out(acc[3])};
}

// ------------------------------------------------------------------ what every kernel does with its sums
__device__ __forceinline__ float silu(float v) {
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}

__device__ __forceinline__ void activate(float (&v)[8], int act) {  // (act: of a known value, or uniform)
  if (act == GELU) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = gelu(v[k]);
  } else if (act == SILU) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = silu(v[k]);
  }
}

// A token of a set: its batch element and its row there.
struct Place {
  uint32_t b, n;
};
__device__ __forceinline__ Place place_of(const Set& s, uint32_t at) {
  uint32_t n = min(at, s.tokens - 1), b = 0;
  if (s.tokens > s.rows) b = n / s.rows, n -= b * s.rows;  // (one batch element: no division)
  return {b, n};
}

// Values p[0 .. 7] of channels c .. c + 7, those of them that there are.
__device__ __forceinline__ u32x4 load8(const uint16_t* p, int c, int columns) {
  if (c + 8 <= columns) return *(const any_u32x4*)p;
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 7; ++k)
    if (c + k < columns) v[k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
  return v;
}

// Eight values of channels c .. c + 7 to `out`, those of them that there are.  (A row that begins between words takes a
// word-aligned 12 bytes and two ends: 16-byte stores across words are slower.)
__device__ __forceinline__ void store8(const Args& a, uint16_t* out, int c, const u32x4& v) {
  typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint32_t words3 __attribute__((ext_vector_type(3), aligned(4)));
  if (c + 8 <= a.columns) {
    if (a.vectors) {
      __builtin_nontemporal_store(v, (u32x4*)out);
    } else if ((uintptr_t)out & 2) {
      out[0] = (uint16_t)v[0];
      *(words3*)(out + 1) = words3{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16};
      out[7] = (uint16_t)(v[3] >> 16);
    } else {
      *(words4*)out = v;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < a.columns) out[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
  }
}

// What a token's eight channels need from memory besides their sums.
struct Epilogue {
  uint16_t* out;
  u32x4 residual, gate;
};

// (c: the first channel; nothing is read where there are none)
__device__ __forceinline__ Epilogue ask(const Args& a, const Set& s, uint32_t at, int c) {
  const Place p = place_of(s, at);
  Epilogue e = {s.out + p.b * s.out_b + (int64_t)p.n * s.out_n + c, {}, {}};
  if (c < a.columns) {
    if (s.residual) e.residual = load8(s.residual + p.b * s.r_b + (int64_t)p.n * s.r_n + c, c, a.columns);
    if (s.gate) e.gate = load8(s.gate + p.b * s.g_b + c, c, a.columns);
  }
  return e;
}

// v: the sums with their bias.
template <bool F16>
__device__ __forceinline__ void finish8(const Args& a, const Set& s, float (&v)[8], const Epilogue& e, uint32_t at, int c) {
  activate(v, a.act);
  if (s.gate) {
    float g[8];
    unpack8<F16>(e.gate, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= g[k];
  }
  if (s.residual) {
    float r[8];
    unpack8<F16>(e.residual, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += r[k];
  }
  if (at < s.tokens) store8(a, e.out, c, pack8<F16>(v));
}

// Rows and columns of the sums of a layer's parts.
__device__ __forceinline__ uint32_t all_tokens(const Args& a) { return a.set[0].tokens + a.set[1].tokens; }
__device__ __forceinline__ uint32_t padded_columns(const Args& a) { return (uint32_t)(a.columns + 7) & ~7u; }

// A workgroup's tile and part of the features.  An XCD has a run of the tiles of one part after another, so that its L2
// serves as few rows and features as can be (all parts of a run of tiles: 512 x 12288 -> 3072 57.8 us, so 55.4; 2048 x
// 12288 -> 1024 65.9 / 60.2).
struct Share {
  uint32_t part, tile;
};
__device__ __forceinline__ Share share_of(const Args& a) {
  const uint32_t at = (blockIdx.x & 7) * a.tiles_xcd + (blockIdx.x >> 3), part = a.splits > 1 ? at / a.tiles : 0;
  return {part, at - part * a.tiles};
}

// The epilogue's bias of a tile's channels, in LDS.
template <bool F16, int TC>
__device__ __forceinline__ void load_bias(const Args& a, const Set& s, int c0, float (&bias)[TC]) {
  const int i = threadIdx.x;
  if (i < TC) bias[i] = s.bias ? to_f<F16>(s.bias[min(c0 + i, a.columns - 1)]) : 0.f;
}

// Where rows end.  A stage is 64 features, 128 bytes: what a lane's load asks for past the row (a multiple of 16 bytes)
// is moved outside the buffer, from where a load brings zeros and reads nothing.
struct RowEnd {
  int full, beyond;  // whole stages, and what the stage after them adds to this lane's offset
  __device__ RowEnd(int features, int chunk)
      : full(features >> 6), beyond(chunk * 8 < (features & 63) ? 0 : (int)0x80000000) {}
  __device__ void stop(int stage) {  // nothing from this stage on
    if (stage <= full) full = stage, beyond = (int)0x80000000;
  }
  __device__ int past(int stage) const {
    return stage < full ? 0 : stage == full ? beyond : (int)0x80000000;
  }
};

// ------------------------------------------------------------------ many rows
// 256 channels x 256 tokens a workgroup of four waves, 128 x 128 each; one workgroup a CU, which walks its tiles.
//  * Two stages of 64 KB in LDS, 64 features of every row (a row's 128 bytes are one request to the L2), by direct loads.
//  * A stage's two steps of 32 features each have registers of their own.  Everyone has read a stage when a quarter of its
//    products are done, and its place takes the stage after the next from then on: a load has at least 100 products' time
//    until it is waited for, enough for one that misses the L2.
//  * What is asked of memory and LDS is spread among the products: asked for together it holds up their issue.
//  * The stages of consecutive tiles follow one another; what comes after a tile's sums works in registers while the next
//    tile's first stages arrive.
//  * An XCD takes a run of the tiles, four token tiles by all channel tiles at a time, so that its L2 serves both
//    operands.
// Bound by power: the clock falls with what the matrix pipes do, and products of 16 x 16 x 32 take less of it than those of
// 32 x 32 x 16 (16384 x 12288 -> 3072 897 and 942 us).  By machine, that size with residual and gate takes 837 to 905 us,
// 1.37 to 1.48 PFLOP/s, where the library's product alone takes 806 to 839; 8192 x 3072 -> 12288 with GELU 441 to 473 (442);
// 512 and 4096 rows, 3072 -> 9216, 205 to 220.
constexpr int WIDE = 256, WIDE_BAND = 4, WIDE_WAVES = 4;
constexpr int WIDE_STAGE = 2 * WIDE * 128;                  // 64 KB
constexpr int WIDE_LOADS = WIDE_STAGE / 1024 / WIDE_WAVES;  // 1 KB loads of a wave and stage

// What the epilogue does.  All up to GATED are for tiles of one batch element each and work on the sums in registers, with
// EDGE also where tiles are not whole; their columns are a multiple of eight and outputs aligned.  ANY takes any tile
// through LDS (4173 x 3072 -> 9216 238 us, with EDGE 200; 9000 x 1024 -> 9000 with residual and gate 320, 227), and PARTS,
// for a part of the features of any tile, stores the sums themselves.  (One kernel for several kinds of tile keeps too much
// in registers.)
enum Mode { PLAIN, ACT_GELU, ACT_SILU, RESIDUAL, GATED, ANY, PARTS };

// A wave's 128 x 128 sums: acc[i][j] are channels 16 i + 4 (lane / 16) .. + 3 of token 16 j + lane % 16.
struct Sums {
  f32x4 v[8][8];
};

// Four words of two neighbouring 16-channel blocks of a token, four channels of each, exchanged among the four lanes of a
// token so that each has eight channels in a row: chunk 2 (q % 2) + q / 2 of the blocks' four, q = lane / 16.  Undoes
// itself.
__device__ __forceinline__ u32x4 cross(const u32x4& v) {
  const auto lo = __builtin_amdgcn_permlane16_swap(v[0], v[2], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(v[1], v[3], false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
}

// Chunks of two such pairs of blocks, `a` of channels 0 .. 31 and `b` of 32 .. 63 of tokens 0 .. 15, exchanged among lanes 8
// apart so that eight lanes have the 64 channels of a token, tokens 0 .. 7 in a and 8 .. 15 in b.  Undoes itself.
__device__ __forceinline__ void halves(u32x4& a, u32x4& b) {
  const bool upper = threadIdx.x & 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t other = moved_bits<0x128>(upper ? a[k] : b[k]);  // (of the lane 8 on, around 16)
    if (upper) a[k] = other;
    else b[k] = other;
  }
}

// The epilogue of a whole tile of one batch element, a wave's part: tokens from t0 and channels from c0 on; `bias` and
// `gate` are theirs, in LDS.  A store moves 128 bytes, whole lines, of 8 rows (64 of 16 rows: 16384 x 3072 x 12288 892
// us, so 867).
template <bool F16, int MODE, bool EDGE>
__device__ __forceinline__ void finish_wide(const Args& a, const Set& s, const Sums& acc, const float* bias, const float* gate, int c0,
                                            uint32_t t0) {
  constexpr bool ADD = MODE == RESIDUAL || MODE == GATED;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (or addresses stay in registers from tile to tile)
  const int q = lane >> 4, c = c0 + (lane >> 3 & 1) * 32 + (q & 1) * 16 + (q >> 1) * 8;
  const Place p = place_of(s, EDGE ? t0 : t0 + (lane & 7));
  const int64_t n = EDGE ? p.n + (lane & 7) : p.n;
  uint16_t* const out = s.out + p.b * s.out_b + n * s.out_n + c;
  const uint16_t* const from = s.residual + p.b * s.r_b + n * s.r_n + c;
  const int rows = EDGE ? (int)(s.tokens - min(t0, s.tokens)) - (lane & 7) : 0;  // (from this lane's first on)
  constexpr int AHEAD = 2;
  u32x4 res[AHEAD + 1][4] = {};
  auto ask = [&](int j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4& to = res[j % (AHEAD + 1)][i];
      const int row = j * 16 + (i & 1) * 8, across = (i >> 1) * 64;
      if (!EDGE || (row < rows && c + across < a.columns)) to = *(const any_u32x4*)(from + row * s.r_n + across);
    }
  };
  if (ADD) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ask(j);
  }
  f32x4 b[8], g[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    b[i] = *(const f32x4*)(bias + i * 16 + q * 4);
    if (MODE == GATED) g[i] = *(const f32x4*)(gate + i * 16 + q * 4);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (ADD && j + AHEAD < 8) ask(j + AHEAD);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 64 channels
      u32x4* const r = &res[j % (AHEAD + 1)][2 * h];
      if (ADD) halves(r[0], r[1]);
      u32x4 packed[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {  // 32 channels
        const int i = 4 * h + 2 * m;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = moved_out(acc.v[i + (k >> 2)][j][k & 3]) + b[i + (k >> 2)][k & 3];
        activate(v, MODE == ACT_GELU ? GELU : MODE == ACT_SILU ? SILU : NONE);
        if (ADD) {
          float add[8];
          unpack8<F16>(cross(r[m]), add);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = (MODE == GATED ? v[k] * g[i + (k >> 2)][k & 3] : v[k]) + add[k];
        }
        packed[m] = cross(pack8<F16>(v));
      }
      halves(packed[0], packed[1]);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int row = j * 16 + m * 8;
        if (!EDGE || (row < rows && c + h * 64 < a.columns))
          __builtin_nontemporal_store(packed[m], (u32x4*)(out + row * s.out_n + h * 64));
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (all at once take more registers than there are)
  }
}

// The epilogue of any tile: a wave's 32 tokens from t0 on and 128 channels from c0 on, whose sums lie in `box`, the
// wave's sixteen pieces of 1 KB, 4 KB apart.  They come back as four tokens of 16 lanes each.
template <bool F16>
__device__ __forceinline__ void finish_any(const Args& a, const Set& s, const float* bias, int c0, uint32_t t0, const int8_t* box) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (as above)
  const int c = (lane & 15) * 8;
  if (c0 + c >= a.columns) return;
  f32x4 b[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) b[g] = *(const f32x4*)(bias + c + 4 * g);
  Epilogue next = ask(a, s, t0 + (lane >> 4), c0 + c);  // (asked for four tokens ahead)
#pragma unroll 1
  for (int q = 0; q < 8; ++q) {
    const Epilogue now = next;
    const int token = q * 4 + (lane >> 4);
    if (q < 7) next = ask(a, s, t0 + token + 4, c0 + c);
    float v[8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const f32x4 sum = *(const f32x4*)(box + (token >> 1) * 4096 + (token & 1) * 512 + (((lane & 15) ^ (token & 15)) + 16 * g) * 16) + b[g];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * g + k] = sum[k];
    }
    finish8<F16>(a, s, v, now, t0 + token, c0 + c);
  }
}

// The sums of 32 of a wave's tokens, blocks j and j + 1, to its box.  (Units of four channels: even ones in the first half
// of a token's 512 bytes, odd ones in the second, in an order of the token's, so that neither the lanes that write together
// nor those that read together share a bank.)
template <int J>
__device__ __forceinline__ void fill_box(const Sums& acc, int8_t* box) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (as above)
  const int q = lane >> 4, token = lane & 15;
  int8_t* const to = box + (token >> 1) * 4096 + (token & 1) * 512 + (q & 1) * 256;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) *(f32x4*)(to + j * 8 * 4096 + ((i * 2 + (q >> 1)) ^ token) * 16) = moved_out(acc.v[i][J + j]);
}

// A wave's sums of a part of a tile, from channel c0 and token t0 on, for join_kernel.
__device__ __forceinline__ void keep_sums(const Args& a, uint32_t part, int set, const Sums& acc, int c0, uint32_t t0) {
  const int lane = threadIdx.x & 63, c = c0 + (lane >> 4) * 4, across = padded_columns(a);
  const uint32_t tokens = a.set[set].tokens;
  t0 += lane & 15;
  float* const to = a.sums + ((int64_t)part * all_tokens(a) + (set ? a.set[0].tokens : 0) + t0) * across + c;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f32x4 v = moved_out(acc.v[i][j]);
      if (t0 + j * 16 < tokens && c + i * 16 < across) *(f32x4*)(to + (int64_t)j * 16 * across + i * 16) = v;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <bool F16, int MODE, bool EDGE = false>
__global__ __launch_bounds__(64 * WIDE_WAVES, 1) void linear_wide_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) int8_t lds0[WIDE_STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds1[WIDE_STAGE];
  __shared__ __attribute__((aligned(16))) float bias[2][WIDE], gate[2][WIDE];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), row = lane & 15, quarter = lane >> 4;
  const int wc = wave & 1, wt = wave >> 1;
  constexpr bool WHOLE = MODE < ANY && !EDGE;
  const Share mine = MODE == PARTS ? share_of(a) : Share{};
  const int start = mine.part * a.stages_each;
  const int stop = MODE == PARTS ? min(start + a.stages_each, (a.features + 63) / 64) : (a.features + 63) / 64;
  const int stages = max((stop - start + 1) / 2 * 2, 4);  // (an even number)
  // (workgroups go to the eight XCDs in turn)
  const uint32_t first = MODE == PARTS ? mine.tile : (blockIdx.x & 7) * a.tiles_xcd, stride = gridDim.x >> 3;
  uint32_t slot = MODE == PARTS ? 0 : blockIdx.x >> 3;
  if (MODE == PARTS && mine.part >= (uint32_t)a.splits) return;
  if (slot >= a.tiles_xcd || first + slot >= a.tiles) return;
  // Loads: a wave's load j fills LDS rows 8 (4 j + wave) .. + 7, eight lanes a row; rows below WIDE are
  // channels, the others tokens (rows past the operands' ends: the last ones again).  The lane at slot p of
  // row r loads chunk p ^ (r / 2 % 8), so that the chunks that 16 rows' lanes read together lie in
  // different banks.
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  RowEnd ends(a.features, chunk);
  if (MODE == PARTS) ends.stop(stop);
  const int8_t *wbase, *xbase;
  int offset[WIDE_LOADS];
  int aimed = -1;  // the set that `offset` is of
  auto aim = [&](const Tile& t) {
    const Set& s = a.set[t.set];
    const Place begin = place_of(s, t.t0);
    wbase = uniform_pointer((const int8_t*)(s.w + t.c0 * s.w_n));
    xbase = uniform_pointer((const int8_t*)(s.x + begin.b * s.x_b + begin.n * s.x_n));
    if (WHOLE && aimed == t.set) return;  // (whole tiles differ by where they begin)
    aimed = t.set;
#pragma unroll
    for (int j = 0; j < WIDE_LOADS; ++j) {
      const int r = 8 * (WIDE_WAVES * j + wave) + (lane >> 3);
      if (j < WIDE_LOADS / 2) {
        offset[j] = (WHOLE ? r : min(r, a.columns - 1 - t.c0)) * (int)s.w_n * 2 + chunk * 16;
      } else if (WHOLE) {
        offset[j] = (r - WIDE) * (int)s.x_n * 2 + chunk * 16;
      } else {
        const Place p = place_of(s, t.t0 + (r - WIDE));
        offset[j] = (int)(((p.b - begin.b) * s.x_b + ((int64_t)p.n - begin.n) * s.x_n) * 2) + chunk * 16;
      }
    }
  };
  auto load = [&](int8_t* dst, int stage, int j, int past) {
    load_lds16(j < WIDE_LOADS / 2 ? wbase : xbase, dst + 1024 * (WIDE_WAVES * j + wave), offset[j] | past, uniform((start + stage) * 128));
  };
  auto past = [&](int stage) { return ends.past(start + stage); };
  // Operands: lane l holds bytes 16 (l / 16) .. + 15 of a 64-byte step of row l % 16.
  const int read = row * 128 + ((row >> 1 & 7) ^ quarter) * 16;
  u32x4 w[2][8], x[2][8];
  // (k of sixteen, as the products need them)
  auto fetch = [&](const int8_t* src, int u, int k) {
    const int at = read ^ (u * 64);
    if (k == 0 || k > 8) {
      const int j = k ? k - 8 : 0;
      x[u][j] = *(const u32x4*)(src + (WIDE + wt * 128 + j * 16) * 128 + at);
    } else {
      w[u][k - 1] = *(const u32x4*)(src + (wc * 128 + (k - 1) * 16) * 128 + at);
    }
  };
  Sums acc;
  // The 128 products of the stage in `cur`, whose first step is in registers or on its way there; the first step of the one
  // in `next` is fetched (at a tile's end the epilogue needs the registers), and `after` is asked for into `cur`.
  constexpr std::false_type no;
  constexpr std::true_type yes;
  auto step = [&](auto first_one, auto last, int8_t* cur, int8_t* next, int after) {
    constexpr bool FIRST = decltype(first_one)::value, LAST = decltype(last)::value;
    const int after_past = past(uniform(after));
    auto product = [&](auto index) {
      constexpr int k = decltype(index)::value, u = k >> 6, j = k >> 3 & 7, i = k & 7;
      if (FIRST && u == 0) begin16<F16>(w[u][i], x[u][j], acc.v[i][j]);
      else accumulate16<F16>(w[u][i], x[u][j], acc.v[i][j]);
      __builtin_amdgcn_sched_barrier(0);
      if (k < 16) fetch(cur, 1, k);
      if (k == 29) {
        wait_loads<63>();
        barrier();  // nobody reads `cur` any more
      }
      if (!(LAST && MODE == ANY) && k >= 30 && (k - 30) % 6 == 0 && (k - 30) / 6 < WIDE_LOADS) load(cur, after, (k - 30) / 6, after_past);
      if (k == 86) {
        wait_arrivals<LAST && MODE == ANY ? 0 : 10>();  // (what this stage has asked for by now)
        barrier();                                      // `next` is there
      }
      if (!LAST && k >= 88 && k % 2 == 0 && (k - 88) / 2 < 16) fetch(next, 0, (k - 88) / 2);
      __builtin_amdgcn_sched_barrier(0);
    };
    begin_all(product, std::make_integer_sequence<int, 128>());
  };
  // The epilogue's values of channel c0 + threadIdx.x of a tile.
  auto ask_channel = [&](const Tile& t, uint16_t& b, uint16_t& g) {
    const Set& s = a.set[t.set];
    const int c = min(t.c0 + (int)threadIdx.x, a.columns - 1);
    b = s.bias ? s.bias[c] : 0;
    if (MODE == GATED) g = s.gate[place_of(s, t.t0).b * s.g_b + c];
  };
  Tile t = tile_at<WIDE, WIDE, WIDE_BAND>(a, first + slot);
  aim(t);
  uint16_t bias_value, gate_value;
  if (MODE != PARTS) ask_channel(t, bias_value, gate_value);
#pragma unroll
  for (int j = 0; j < WIDE_LOADS; ++j) load(lds0, 0, j, past(0));
#pragma unroll
  for (int j = 0; j < WIDE_LOADS; ++j) load(lds1, 1, j, past(1));
  wait_loads<WIDE_LOADS>();
  barrier();
  for (int parity = 0;; parity ^= 1) {
    const Tile done = t;
    const Set& s = a.set[done.set];
    if (MODE != PARTS) bias[parity][threadIdx.x] = to_f<F16>(bias_value);  // (read after the next barriers)
    if (MODE == GATED) gate[parity][threadIdx.x] = to_f<F16>(gate_value);
#pragma unroll
    for (int k = 0; k < 16; ++k) fetch(lds0, 0, k);
    step(yes, no, lds0, lds1, 2);
    step(no, no, lds1, lds0, 3);
    for (int n = 4; n < stages; n += 2) {
      step(no, no, lds0, lds1, n);
      step(no, no, lds1, lds0, n + 1);
    }
    slot += stride;
    const bool more = MODE != PARTS && slot < a.tiles_xcd && first + slot < a.tiles;
    if (more) t = tile_at<WIDE, WIDE, WIDE_BAND>(a, first + slot);
    aim(t);  // (after the last tile: its own first stages once more, never multiplied)
    if (MODE != PARTS) ask_channel(t, bias_value, gate_value);  // (before the stores, which a load after them would wait for)
    step(no, no, lds0, lds1, 0);
    step(no, yes, lds1, lds0, 1);
    settle();
    const int c0 = done.c0 + wc * 128;
    const uint32_t t0 = done.t0 + wt * 128;
    if constexpr (MODE == PARTS) {
      keep_sums(a, mine.part, done.set, acc, c0, t0);
    } else if constexpr (MODE < ANY) {
      finish_wide<F16, MODE, EDGE>(a, s, acc, &bias[parity][wc * 128], &gate[parity][wc * 128], c0, t0);
    } else {
      int8_t* const box = lds1 + 1024 * wave;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        if (j == 0) fill_box<0>(acc, box);
        else if (j == 1) fill_box<2>(acc, box);
        else if (j == 2) fill_box<4>(acc, box);
        else fill_box<6>(acc, box);
        finish_any<F16>(a, s, &bias[parity][wc * 128], c0, t0 + j * 32, box);
      }
      wait_loads<63>();  // (into the pieces that this wave's own epilogue has read)
#pragma unroll
      for (int j = 0; j < WIDE_LOADS; ++j) load(lds1, 1, j, past(1));
    }
    if (!more) break;
  }
  wait_loads<0>();  // (nothing may still be on its way to LDS when the workgroup ends)
}

// ------------------------------------------------------------------ fewer rows
// TC channels x TT tokens a workgroup, in tiles so small that most CUs have one.  LDS bounds it: a stage of 64 features of
// 96 x 64 is 20 KB written and 32 KB read, 0.25 us, 80 bytes a ns into a CU (direct loads alone reach 134).  So the loads
// go to LDS past the registers, into a ring of R stages, spread over the products, and where the tiles are fewer than the
// CUs the features are split among workgroups (share_of).  A stage's features are in four parts of 16, a wave each in the
// smallest tiles, or two waves that share the tokens (of 32 tokens: the channels), whose epilogue is shorter.  The sums
// meet in LDS, and a thread finishes eight channels of a token: neighbouring lanes read and write whole lines.  Rows
// past the operands' ends are zeros that nothing reads.  77 x 4096 -> 3072 13.4 us, 23 with the weight from memory; 2048 x
// 2048 -> 2048 (128 x 128) 21, 0.8 PFLOP/s.
// AHEAD > 0: rows at any address, by registers that AHEAD stages are on their way to, then into the ring: 0.3 us a stage of
// 64 x 64, where direct loads take 0.2, but no copies.
template <int TC, int TT, int WAVES>
struct Ring {
  static constexpr int STAGE = (TC + TT) * 128, GROUPS = STAGE / 1024, LOADS = (GROUPS + WAVES - 1) / WAVES;
  static constexpr int CW = TT > 32 ? TC : TC / 2, TW = TT > 32 ? TT / 2 : TT;  // of half the sums
  static constexpr int BOX = TW * CW * 4;
  static constexpr int CF = (WAVES > 4 ? CW : TC) / 32, TF = (WAVES > 4 ? TW : TT) / 32;  // of a wave
};

template <bool F16, int TC, int TT, int R, int WAVES, int AHEAD = 0>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void linear_tile_kernel(Args a) {
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
  __shared__ __attribute__((aligned(16))) float bias[TC];
  auto ring = [&](auto index) -> int8_t* {
    constexpr int i = decltype(index)::value % R;
    return i == 0 ? lds0 : i == 1 ? lds1 : i == 2 ? lds2 : i == 3 ? lds3 : i == 4 ? lds4 : i == 5 ? lds5 : i == 6 ? lds6 : lds7;
  };
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int part = WAVES > 4 ? wave >> 1 : wave, share = WAVES > 4 ? wave & 1 : 0;
  const Share mine = share_of(a);
  if (mine.part >= (uint32_t)a.splits || mine.tile >= a.tiles) return;
  const Tile t = tile_at<TC, TT, 8>(a, mine.tile);
  const Set& s = a.set[t.set];
  load_bias<F16>(a, s, t.c0, bias);
  // Loads as in the wide kernel.
  const Place begin = place_of(s, t.t0);
  const int8_t *wbase = (const int8_t*)(s.w + t.c0 * s.w_n), *xbase = (const int8_t*)(s.x + begin.b * s.x_b + begin.n * s.x_n);
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  int offset[LOADS];  // (of direct loads)
  const uint16_t* row[LOADS];  // (of the others)
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = 8 * (WAVES * j + wave) + (lane >> 3);
    if (AHEAD) {
      const Place p = place_of(s, t.t0 + (r - TC));
      row[j] = r < TC ? s.w + min(t.c0 + r, a.columns - 1) * s.w_n : s.x + p.b * s.x_b + p.n * s.x_n;
    } else if (r < TC) {
      offset[j] = r < a.columns - t.c0 ? r * (int)s.w_n * 2 + chunk * 16 : (int)0x80000000;
    } else {
      const Place p = place_of(s, t.t0 + (r - TC));
      offset[j] = (uint32_t)(r - TC) < s.tokens - t.t0
                      ? (int)(((p.b - begin.b) * s.x_b + ((int64_t)p.n - begin.n) * s.x_n) * 2) + chunk * 16
                      : (int)0x80000000;
    }
  }
  const int first = mine.part * a.stages_each, last = min(first + a.stages_each, (a.features + 63) / 64);
  RowEnd ends(a.features, chunk);
  ends.stop(last);
  const bool all = WAVES * (LOADS - 1) + wave < F::GROUPS;  // (the last loads are not every wave's)
  // (rows at any address: by registers)
  u32x4 held[AHEAD ? AHEAD : 1][LOADS];
  auto ask_rows = [&](u32x4& to, int stage, int j) { to = *(const any_u32x4*)(row[j] + min(stage * 64 + chunk * 8, a.features - 8)); };
  auto hand_in = [&](int8_t* dst, u32x4 v, int stage, int j) {
    if (stage * 64 + 64 > a.features) v = drop_values(v, min(max(stage * 64 + chunk * 8 - (a.features - 8), 0), 8));
    *(u32x4*)(dst + 1024 * (WAVES * j + wave) + lane * 16) = v;
  };
  auto load = [&](int8_t* dst, int stage, int j, int past) {
    const int group = WAVES * j + wave;
    if (F::GROUPS % WAVES == 0 || j < LOADS - 1 || all)
      load_lds16(group * 8 < TC ? wbase : xbase, dst + 1024 * group, offset[j] | past, uniform(stage * 128));
  };
  auto arrivals = [&] {
    if (F::GROUPS % WAVES == 0 || all) wait_arrivals<(R - 3) * LOADS>();
    else wait_arrivals<(R - 3) * (LOADS - 1)>();
  };
  const int read = col * 128 + ((col >> 1 & 7) ^ (2 * part + half)) * 16;
  const int wread = read + (TT > 32 ? 0 : share * CW * 128), xread = read + (TC + (TT > 32 ? share * TW : 0)) * 128;
  u32x4 w[2][CF], x[2][TF];
  auto fetch = [&](const int8_t* src, int to) {
#pragma unroll
    for (int i = 0; i < CF; ++i) w[to][i] = *(const u32x4*)(src + wread + i * 4096);
#pragma unroll
    for (int j = 0; j < TF; ++j) x[to][j] = *(const u32x4*)(src + xread + j * 4096);
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x16 acc[TF][CF] = {};
  // Stage n's operands are in w, x, or on their way; stage n + 1 is in LDS.  The stage whose reads ended in
  // the last step takes n + R - 1.  Before the barrier stage n + 2 is there.
  int n = first;
  auto step = [&](auto index) {
    constexpr int I = decltype(index)::value;
    int8_t* const free = ring(std::integral_constant<int, I + R - 1>());
    const int past = ends.past(uniform(n + R - 1));
    int asked = 0, done = 0;
#pragma unroll
    for (int j = 0; j < TF; ++j)
#pragma unroll
      for (int i = 0; i < CF; ++i) {
        acc[j][i] = multiply32<F16>(w[I & 1][i], x[I & 1][j], acc[j][i]);
        for (++done; asked * TF * CF < done * LOADS; ++asked) {
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (AHEAD) {
            hand_in(free, held[I % AHEAD][asked], n + R - 1, asked);
            ask_rows(held[I % AHEAD][asked], n + R - 1 + AHEAD, asked);
          } else {
            load(free, n + R - 1, asked, past);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    if (AHEAD) wait_loads<63>();  // (what it has written is in LDS)
    fetch(ring(std::integral_constant<int, I + 1>()), ~I & 1);
    if (!AHEAD) arrivals();
    barrier();
    return ++n == last;
  };
  if constexpr (AHEAD) {
    u32x4 now[R - 1][LOADS];
#pragma unroll
    for (int i = 0; i < R - 1 + AHEAD; ++i)
#pragma unroll
      for (int j = 0; j < LOADS; ++j) ask_rows(i < R - 1 ? now[i][j] : held[(i - (R - 1)) % AHEAD][j], first + i, j);
    auto begin_stage = [&](auto index) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) hand_in(ring(index), now[decltype(index)::value][j], first + decltype(index)::value, j);
    };
    begin_all(begin_stage, std::make_integer_sequence<int, R - 1>());
    wait_loads<63>();
  } else {
    // (Zeros into the last stage, so that the compiler, which tracks what is on its way to which array, has met them
    // all before the loop: otherwise it waits for everything each time around.)
    load(ring(std::integral_constant<int, R - 1>()), 0, 0, (int)0x80000000);
    auto begin_stage = [&](auto index) {
      constexpr int I = decltype(index)::value;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load(ring(index), first + I, j, ends.past(first + I));
    };
    begin_all(begin_stage, std::make_integer_sequence<int, R - 1>());
    arrivals();
  }
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
          f32x4* const at = (f32x4*)(box(part & 1, h) + unit(token + col, c + g * 8 + half * 4));
          const f32x4 v = {acc[j][i][4 * g], acc[j][i][4 * g + 1], acc[j][i][4 * g + 2], acc[j][i][4 * g + 3]};
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
    const uint32_t to = t.t0 + token;
    if (to >= s.tokens || t.c0 + c >= a.columns) continue;
    f32x4 sum[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int at = unit(TT > 32 ? token % TW : token, (TT > 32 ? c : c % CW) + 4 * g);
      sum[g] = *(const f32x4*)(box(0, h) + at) + *(const f32x4*)(box(1, h) + at);
    }
    if (a.splits > 1) {
      f32x4* const parts = (f32x4*)(a.sums + ((int64_t)mine.part * all_tokens(a) + (t.set ? a.set[0].tokens : 0) + to) * padded_columns(a) + t.c0 + c);
      parts[0] = sum[0];
      parts[1] = sum[1];
      continue;
    }
    const Epilogue more = ask(a, s, to, t.c0 + c);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = sum[k >> 2][k & 3] + bias[c + k];
    finish8<F16>(a, s, v, more, to, t.c0 + c);
  }
}

// The sums of a layer's parts, in their order, and the epilogue: a thread has eight channels of a token.  Bound by their
// read: eight parts of 512 x 3072, 50 MB, with residual and gate 10.9 us, 5.2 TB/s.
template <bool F16>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  const uint32_t across = padded_columns(a) / 8, tokens = all_tokens(a);
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / across;
  if (row >= tokens) return;
  const int c = (int)(i - row * across) * 8;
  const int set = row >= a.set[0].tokens;
  const Set& s = a.set[set];
  const uint32_t to = row - (set ? a.set[0].tokens : 0);
  const Epilogue more = ask(a, s, to, c);
  const u32x4 bias = s.bias ? load8(s.bias + c, c, a.columns) : u32x4{};
  const f32x4* from = (const f32x4*)(a.sums + (int64_t)row * padded_columns(a) + c);
  const int64_t step = (int64_t)tokens * padded_columns(a) / 4;
  f32x4 sum[2] = {};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k, from += step) {
    sum[0] += from[0];
    sum[1] += from[1];
  }
  float v[8];
  unpack8<F16>(bias, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] += sum[k >> 2][k & 3];
  finish8<F16>(a, s, v, more, to, c);
}

// ------------------------------------------------------------------ a few rows
// 16 channels by up to 16 tokens a workgroup; its eight waves take turns at 128 features, straight from memory into the
// matrix instruction's registers, and their sums meet in LDS.  Rows may lie at any address.  Bound by the weight's
// read: 1 x 3072 -> 18432 25.8 us, 4.4 TB/s (linear_rows_kernel takes 21.2 for one such layer and 16.2 for each of
// seven).
constexpr int FEW_ROWS = 16, FEW_WAVES = 8;

template <bool F16>
__global__ __launch_bounds__(64 * FEW_WAVES) void linear_few_kernel(Args a) {
  __shared__ float sums[FEW_WAVES][16][17];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), r = lane & 15, quarter = lane >> 4;
  const int set = blockIdx.x >= a.tiles0;
  const Set& s = a.set[set];
  const int c0 = (int)(blockIdx.x - (set ? a.tiles0 : 0)) * 16;
  const uint16_t* const w = s.w + min(c0 + r, a.columns - 1) * s.w_n;
  const Place p = place_of(s, r);
  const uint16_t* const x = s.x + p.b * s.x_b + p.n * s.x_n;
  f32x4 acc[2] = {};
  const int whole = a.features & ~127;
  for (int k0 = wave * 128; k0 < whole; k0 += FEW_WAVES * 128) {
    u32x4 wv[4], xv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) wv[u] = __builtin_nontemporal_load((const any_u32x4*)(w + k0 + u * 32 + quarter * 8));
#pragma unroll
    for (int u = 0; u < 4; ++u) xv[u] = *(const any_u32x4*)(x + k0 + u * 32 + quarter * 8);
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u & 1] = multiply16<F16>(wv[u], xv[u], acc[u & 1]);
  }
  if (whole < a.features && wave == whole / 128 % FEW_WAVES) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      acc[u & 1] = multiply16<F16>(load_row8<false>(w, whole + u * 32 + quarter * 8, a.features),
                                   load_row8<false>(x, whole + u * 32 + quarter * 8, a.features), acc[u & 1]);
  }
  // (lane: channels 4 quarter .. + 3 of token r)
#pragma unroll
  for (int k = 0; k < 4; ++k) sums[wave][r][quarter * 4 + k] = acc[0][k] + acc[1][k];
  __syncthreads();
  const int token = threadIdx.x >> 4, c = c0 + (threadIdx.x & 15);
  if (threadIdx.x >= 256 || (uint32_t)token >= s.tokens || c >= a.columns) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < FEW_WAVES; ++k) v += sums[k][token][threadIdx.x & 15];
  if (s.bias) v += to_f<F16>(s.bias[c]);
  if (a.act == GELU) v = gelu(v);
  else if (a.act == SILU) v = silu(v);
  const Place at = place_of(s, token);
  if (s.gate) v *= to_f<F16>(s.gate[at.b * s.g_b + c]);
  if (s.residual) v += to_f<F16>(s.residual[at.b * s.r_b + (int64_t)at.n * s.r_n + c]);
  s.out[at.b * s.out_b + (int64_t)at.n * s.out_n + c] = from_f<F16>(v);
}

// ------------------------------------------------------------------ rows that direct loads cannot take
// Direct loads to LDS bring 16 bytes from a multiple of 16, and a row's last 16 must not reach into what follows.
// Other rows (an odd length, an odd column of a wider buffer) go by registers (ROWS64x64) or, where that would take
// longer, are copied into rows of a multiple of 64 values, zeros after their own: 7000 rows of 5001 39 us, 3.6 TB/s, 999 and 777 rows of 1001 5.1.  Rows that they can take are not copied,
// though 128 bytes of them straddle two lines: 16384 x 5000 -> 5000 729 us, copied 720; 4096 x 5000 -> 4096 151, 150; 2000 x
// 1000 -> 2000 18, 26.
struct PadArgs {
  struct Matrix {
    const uint16_t* from;
    uint16_t* to;
    int64_t b, n;
    uint32_t rows, all;  // rows of a batch element, and of all
  } m[4];
  uint32_t first[5];  // workgroups up to each matrix
  int32_t features, padded;
};

constexpr uint32_t PAD_GROUPS = 1 << 16;

__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs p) {
  for (uint32_t group = blockIdx.x; group < p.first[4]; group += gridDim.x) {
    int i = 0;
    while (group >= p.first[i + 1]) ++i;
    const PadArgs::Matrix& m = p.m[i];
    // a wave a row
    const uint32_t row = (group - p.first[i]) * 4 + (threadIdx.x >> 6);
    if (row >= m.all) continue;
    const uint32_t b = row / m.rows;
    const uint16_t* const from = m.from + b * m.b + (int64_t)(row - b * m.rows) * m.n;
    uint16_t* const to = m.to + (int64_t)row * p.padded;
    for (int c = (threadIdx.x & 63) * 8; c < p.padded; c += 512) *(u32x4*)(to + c) = load_row8<false>(from, c, p.features);
  }
}

// ------------------------------------------------------------------ launches
// (TWO64x64: with half the stages in LDS, so that a CU has two workgroups; ROWS64x64: the same of rows at any address)
enum Kernel { T64x32, T32x64, T64x64, TWO64x64, T96x64, T96x128, T128x128, WIDE256, ROWS64x64, KERNELS, FEW16 = KERNELS };

// A kernel's tile, how many workgroups the card's 256 CUs hold at once, and what its time is made of, in us: the launch, a round of so
// many workgroups, a round's stage of 64 features, what a stage takes longer when all CUs are at it, each megabyte of rows
// and weight, each million outputs, and, in parts, the join and each megabyte of their sums.  Fitted to 4418 times of 424 sizes
// whose operands come from memory, which they meet to 12% (one sigma); some by more, 16384 x 5032 -> 5000 580 for 740 us, where
// the choice is the same.
struct Shape {
  int tc, tt;
  float at_once, launch, round, stage, full, megabyte, outputs, join, sums;
};
constexpr Shape SHAPES[KERNELS] = {
    {64, 32, 256.f, 4.4f, 1.0f, 0.148f, 0.002f, 0.172f, 1.39f, 3.7f, 0.00f},
    {32, 64, 256.f, 3.0f, 2.4f, 0.147f, 0.043f, 0.145f, 1.36f, 3.7f, 0.00f},
    {64, 64, 256.f, 3.4f, 2.3f, 0.196f, 0.063f, 0.153f, 1.09f, 3.3f, 0.28f},
    {64, 64, 512.f, 3.7f, 1.9f, 0.231f, 0.231f, 0.169f, 0.95f, 3.0f, 0.40f},
    {96, 64, 256.f, 3.8f, 3.5f, 0.261f, 0.050f, 0.150f, 1.12f, 2.0f, 0.43f},
    {96, 128, 256.f, 5.9f, 3.6f, 0.400f, 0.033f, 0.130f, 1.40f, 0.9f, 0.51f},
    {128, 128, 256.f, 8.0f, 2.7f, 0.454f, 0.058f, 0.128f, 1.57f, 0.0f, 0.48f},
    {256, 256, 256.f, 5.6f, 1.5f, 1.133f, 0.081f, 0.085f, 0.82f, 3.9f, 0.36f},
    {64, 64, 512.f, 2.4f, 4.3f, 0.270f, 0.345f, 0.236f, 0.60f, 2.9f, 0.81f},
};
constexpr float WIDE_ANY_ROUND = 22.f;               // (through LDS; fitted to 180 sizes of that epilogue)
constexpr float COPY = 4.3f, COPY_MEGABYTE = 0.116f;  // (of rows that are copied first, read and written)

// Tiles of TC x TT of both sets.
int64_t tiles_of(const Args& a, int count, int tc, int tt) {
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i)
    tiles += ((a.set[i].tokens + (int64_t)tt - 1) / tt) * ((a.columns + (int64_t)tc - 1) / tc);
  return tiles;
}

struct Choice {
  Kernel kernel;
  int splits;
  float us;
};

int64_t sums_bytes(const Args& a, int splits) {
  return splits > 1 ? (int64_t)splits * ((int64_t)a.set[0].tokens + a.set[1].tokens) * ((a.columns + 7) & ~7) * 4 : 0;
}

// Whether all of the wide kernel's tiles are whole, of one batch element and stored in 16 bytes.
bool whole_tiles(const Args& a, int count) {
  bool whole = a.vectors && a.columns % WIDE == 0;
  for (int i = 0; i < count; ++i) whole &= a.set[i].rows % WIDE == 0;
  return whole;
}

// Whether each of its tiles lies in one batch element, and all outputs are stored in 16 bytes.
bool one_element(const Args& a, int count) {
  bool one = a.vectors && a.columns % 8 == 0;
  for (int i = 0; i < count; ++i) one &= a.set[i].tokens == a.set[i].rows || a.set[i].rows % WIDE == 0;
  return one;
}

// The wide kernel's epilogue for these sets.
Mode mode_of(const Args& a, int count) {
  const bool residual = a.set[0].residual, gate = a.set[0].gate;
  bool same = one_element(a, count);
  for (int i = 0; i < count; ++i) same &= residual == !!a.set[i].residual && gate == !!a.set[i].gate;
  if (!same || (a.act != NONE && residual)) return ANY;
  return a.act == GELU ? ACT_GELU : a.act == SILU ? ACT_SILU : gate ? GATED : residual ? RESIDUAL : PLAIN;
}

// What a kernel takes for the sets, in us.
float estimate(const Args& a, int count, Kernel k, int splits) {
  const Shape& s = SHAPES[k];
  const float rounds = (float)(tiles_of(a, count, s.tc, s.tt) * splits) / s.at_once, whole = std::floor(rounds), rest = rounds - whole;
  const float stages = (float)(((a.features + 63) / 64 + splits - 1) / splits);
  const float round = k == WIDE256 && splits == 1 && mode_of(a, count) == ANY ? WIDE_ANY_ROUND : s.round;
  const float tokens = (float)a.set[0].tokens + (float)a.set[1].tokens, rows = tokens + (float)count * (float)a.columns;
  float us = s.launch + whole * (round + stages * (s.stage + s.full)) +
             (rest > 0.f ? round + stages * (s.stage + s.full * rest * rest) : 0.f) + s.megabyte * 2e-6f * rows * (float)a.features +
             s.outputs * 1e-6f * tokens * (float)a.columns;
  if (splits > 1) us += s.join + s.sums * 1e-6f * (float)sums_bytes(a, splits);
  return us;
}

// The same of linear_few_kernel: a wave's way through the features, or the read of the weights; both are slower for rows that
// begin between 16 bytes.  What bounds a few rows, it / the others, us: 1 x 3072 -> 4096 8.2 / 11.6, 16 rows of it 9.7 / 12.4;
// many features, 8 x 12288 -> 512 25.1 / 11.4 (in parts), or the weights of more rows, 16 x 3072 -> 9216 22.9 / 17.4, 8 x 14633
// -> 9216 176 / 132.
float estimate_few(const Args& a, int count, bool aligned) {
  const float tokens = (float)std::max(a.set[0].tokens, a.set[1].tokens), slower = aligned ? 1.f : 1.6f + 0.05f * tokens;
  const float megabytes = 2e-6f * (float)count * (float)a.columns * (float)a.features;
  return std::max(2.3f + (float)a.features / 1024.f * (1.65f + 0.027f * tokens) * slower,
                  3.f + megabytes * (0.25f + 0.007f * tokens) * slower);
}

// The kernel, and the parts that it takes the features in, of the least estimate.  Parts pay where few tiles leave CUs idle
// over many features; they are tried while all their workgroups fit the card at once, with four stages each or more.
// Measured, the best of one part / the parts: 99 x 8472 -> 64 30.4 / 9.9 us, 512 x 12288 -> 3072 72.8 / 60 (eight of the
// wide kernel), 1280 x 13824 -> 5120 251 / 171 (two of it).  Over 264 sizes the choice takes 1.6% more time than the best of
// all; the best of one part takes 13.9% more over 175 of them.  What the wide kernel's epilogue is counts: over 100 sizes
// with an activation and a residual the choice takes 2.5% more than the best, and 29% as if it were in registers (1330 x 64
// -> 1664 8.9 / 34.9 us, 10240 x 128 -> 256 9.7 / 36.2); over 80 of several batch elements or odd columns 0.8%.  TWO64x64
// pays where many tiles are short: the best of the others / with it 5993 x 128 -> 2752 47.5 / 39.5, 4576 x 64 -> 960 16.6 /
// 12.8, 657 x 1216 -> 2624 16.2 / 13.7; alone on its CU it is slower (77 x 4096 -> 3072 27.6, T64x64 21.9); without it the
// choice takes 5.8% more than the best.  Rows that direct loads cannot take are copied, or not, by the same measure. Copied
// / as they are: 999 x 1001 -> 777 14.0 / 11.7 us, 2405 x 13 -> 20 11.0 / 7.2, 64 x 12001 -> 17000 262 / 219, 2000 x 5001
// -> 5000 144 / 345; over 160 such sizes the choice takes 1.0% more than the better one, copies alone 27%.
Choice choose(const Args& a, int count, int first, int last) {
  Choice best = {(Kernel)last, 1, estimate(a, count, (Kernel)last, 1)};
  const int stages = (a.features + 63) / 64;
  for (int i = first; i <= last; ++i) {
    const Kernel k = (Kernel)i;
    const int64_t tiles = tiles_of(a, count, SHAPES[k].tc, SHAPES[k].tt);
    if (tiles >= (1 << 21)) continue;  // (a grid holds fewer than 2^32 threads)
    for (int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (splits > 1 && (tiles * splits > 256 || stages < 4 * splits)) break;
      const float us = estimate(a, count, k, splits);
      if (us < best.us) best = {k, splits, us};
    }
  }
  return best;
}

template <bool F16, bool EDGE>
void launch_wide(const Args& a, Mode mode, const dim3& grid, hipStream_t st) {
  const dim3 block(64 * WIDE_WAVES);
  switch (mode) {
    case PLAIN: hipLaunchKernelGGL((linear_wide_kernel<F16, PLAIN, EDGE>), grid, block, 0, st, a); break;
    case ACT_GELU: hipLaunchKernelGGL((linear_wide_kernel<F16, ACT_GELU, EDGE>), grid, block, 0, st, a); break;
    case ACT_SILU: hipLaunchKernelGGL((linear_wide_kernel<F16, ACT_SILU, EDGE>), grid, block, 0, st, a); break;
    case RESIDUAL: hipLaunchKernelGGL((linear_wide_kernel<F16, RESIDUAL, EDGE>), grid, block, 0, st, a); break;
    case GATED: hipLaunchKernelGGL((linear_wide_kernel<F16, GATED, EDGE>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((linear_wide_kernel<F16, ANY>), grid, block, 0, st, a);
  }
}

template <bool F16>
int launch_kernel(Args& a, int count, const Choice& choice, hipStream_t st) {
  const int tc = SHAPES[choice.kernel].tc, tt = SHAPES[choice.kernel].tt, stages = (a.features + 63) / 64;
  const int64_t tiles = tiles_of(a, count, tc, tt);
  HB_REQUIRE(tiles < (1ll << 30), "too many output tiles for one launch");
  a.channel_tiles = (uint32_t)((a.columns + tc - 1) / tc);
  a.tiles0 = (uint32_t)tiles_of(a, 1, tc, tt);
  a.tiles = (uint32_t)tiles;
  a.stages_each = (stages + choice.splits - 1) / choice.splits;
  if (choice.kernel == WIDE256) a.stages_each = (a.stages_each + 1) & ~1;  // (which it takes in twos)
  a.splits = (stages + a.stages_each - 1) / a.stages_each;
  a.tiles_xcd = (a.tiles * a.splits + 7) / 8;
  const dim3 each(8 * a.tiles_xcd), four(256), eight(512);
  switch (choice.kernel) {
    case T64x32: hipLaunchKernelGGL((linear_tile_kernel<F16, 64, 32, 6, 4>), each, four, 0, st, a); break;
    case T32x64: hipLaunchKernelGGL((linear_tile_kernel<F16, 32, 64, 8, 4>), each, four, 0, st, a); break;
    case T64x64: hipLaunchKernelGGL((linear_tile_kernel<F16, 64, 64, 8, 8>), each, eight, 0, st, a); break;
    case TWO64x64: hipLaunchKernelGGL((linear_tile_kernel<F16, 64, 64, 4, 8>), each, eight, 0, st, a); break;
    case T96x64: hipLaunchKernelGGL((linear_tile_kernel<F16, 96, 64, 7, 8>), each, eight, 0, st, a); break;
    case T96x128: hipLaunchKernelGGL((linear_tile_kernel<F16, 96, 128, 5, 8>), each, eight, 0, st, a); break;
    case T128x128: hipLaunchKernelGGL((linear_tile_kernel<F16, 128, 128, 4, 8>), each, eight, 0, st, a); break;
    case ROWS64x64: hipLaunchKernelGGL((linear_tile_kernel<F16, 64, 64, 4, 8, 4>), each, eight, 0, st, a); break;
    default: {
      const uint32_t per_xcd = std::max(1, device_cu_count() / 8);
      const dim3 grid(8 * std::min(a.tiles_xcd, per_xcd)), block(64 * WIDE_WAVES);
      if (a.splits > 1) hipLaunchKernelGGL((linear_wide_kernel<F16, PARTS>), each, block, 0, st, a);
      else if (whole_tiles(a, count)) launch_wide<F16, false>(a, mode_of(a, count), grid, st);
      else launch_wide<F16, true>(a, mode_of(a, count), grid, st);
    }
  }
  HB_HIP(hipGetLastError());
  if (a.splits > 1) {
    const int64_t threads = (int64_t)(a.set[0].tokens + a.set[1].tokens) * ((a.columns + 7) / 8);
    hipLaunchKernelGGL((join_kernel<F16>), dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, st, a);
    HB_HIP(hipGetLastError());
  }
  return HB_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Whether direct loads take a matrix of `features` columns: rows of whole 16 bytes, and 256 of them, in order, within
// what a load's offset reaches (2^31 bytes, the row itself among them).
bool direct(const void* p, int64_t batch, int64_t rows, int64_t b, int64_t n, int32_t features) {
  if (features % 8 || !aligned16(p) || (rows > 1 && n % 8) || (batch > 1 && b % 8)) return false;
  const int64_t last = (rows - 1) * n;
  if (batch > 1 && b < last) return false;  // (a later row would lie before a tile's first)
  const int64_t batches = std::min(batch - 1, 255 / rows + 1);
  return (batches * b + std::min<int64_t>(255, rows - 1) * n) * 2 + features * 2ll < (1ll << 31) - 4096;
}

int64_t padded_bytes(int64_t rows, int32_t features) { return rows * ((features + 63ll) / 64 * 64) * 2; }

constexpr int MAX_DEPTH = 1 << 20;
constexpr int MAX_COLUMNS = 1 << 25;  // (few rows of two sets: 32 threads a channel, and a grid holds fewer than 2^32)

// A call, and what it takes: the launches and the workspace.
struct Plan {
  Args a;
  PadArgs pad;
  Choice choice;
  int copies;
  int64_t bytes;  // of copied rows, and of all
};

int plan(Plan& p, int32_t count, int32_t batch, const int32_t* rows, int32_t columns, int32_t features, int32_t act,
         void* const* pointers, const int64_t* strides, void* workspace) {
  HB_REQUIRE(count == 1 || count == 2, "count must be 1 or 2");
  HB_REQUIRE(rows && pointers && strides, "null pointer argument");
  HB_REQUIRE(columns > 0 && columns <= MAX_COLUMNS, "columns must be in [1, %d] (got %d)", MAX_COLUMNS, columns);
  HB_REQUIRE(features > 0 && features <= MAX_DEPTH, "features must be in [1, %d] (got %d)", MAX_DEPTH, features);
  p = {};
  Args& a = p.a;
  a.columns = columns;
  a.features = features;
  a.act = act;
  a.vectors = 1;
  bool few = true;
  for (int i = 0; i < count; ++i) {
    HB_REQUIRE(batch > 0 && rows[i] > 0 && (int64_t)batch * rows[i] < (1ll << 31), "batch and rows must be positive, with fewer than 2^31 rows in all");
    few &= (int64_t)batch * rows[i] <= FEW_ROWS;
  }
  bool copied[2][2] = {};
  float megabytes = 0.f;
  p.pad.features = features;
  p.pad.padded = (features + 63) / 64 * 64;
  for (int i = 0; i < count; ++i) {
    void* const* q = pointers + 6 * i;
    const int64_t* st = strides + 8 * i;
    HB_REQUIRE(q[0] && q[1] && q[5], "null pointer argument");
    HB_REQUIRE(!q[4] || q[3], "a gate needs its residual");
    for (int k = 0; k < 6; ++k) HB_REQUIRE(((uintptr_t)q[k] & 1) == 0, "every pointer must be 2-byte aligned");
    for (int k = 0; k < 8; ++k) HB_REQUIRE(st[k] >= 0, "strides must be non-negative");
    Set& s = a.set[i];
    s = {(const uint16_t*)q[0], (const uint16_t*)q[1], (const uint16_t*)q[2], (const uint16_t*)q[3], (const uint16_t*)q[4],
         (uint16_t*)q[5], st[0], st[1], st[2], st[3], st[4], st[5], st[6], st[7], (uint32_t)rows[i], (uint32_t)(batch * rows[i])};
    a.vectors &= aligned16(s.out) && s.out_b % 8 == 0 && s.out_n % 8 == 0;
    copied[i][0] = !direct(s.x, batch, rows[i], s.x_b, s.x_n, features);
    copied[i][1] = !direct(s.w, 1, columns, 0, s.w_n, features);
    megabytes += 2e-6f * (float)(features + p.pad.padded) * ((copied[i][0] ? (float)s.tokens : 0.f) + (copied[i][1] ? (float)columns : 0.f));
  }
  p.choice = choose(a, count, T64x32, WIDE256);
  if (megabytes > 0.f) {
    p.choice.us += COPY + COPY_MEGABYTE * megabytes;
    if (features >= 8 && tiles_of(a, count, 64, 64) < (1 << 21)) {
      const Choice as_they_are = choose(a, count, ROWS64x64, ROWS64x64);
      if (as_they_are.us < p.choice.us) p.choice = as_they_are;
    }
  }
  if (few && estimate_few(a, count, megabytes == 0.f) < p.choice.us) p.choice = {FEW16, 1};
  if (p.choice.kernel < ROWS64x64) {
    auto copy = [&](const uint16_t*& from, int64_t& b, int64_t& n, uint32_t rows_of_one, uint32_t all) {
      uint16_t* const to = (uint16_t*)((char*)workspace + p.bytes);
      p.bytes += padded_bytes(all, features);
      p.pad.m[p.copies] = {from, to, b, n, rows_of_one, all};
      p.pad.first[p.copies + 1] = p.pad.first[p.copies] + (all + 3) / 4;
      ++p.copies;
      from = to;
      n = p.pad.padded;
      b = n * rows_of_one;
    };
    int64_t none = 0;
    for (int i = 0; i < count; ++i) {
      Set& s = a.set[i];
      if (copied[i][0]) copy(s.x, s.x_b, s.x_n, s.rows, s.tokens);
      if (copied[i][1]) copy(s.w, none, s.w_n, (uint32_t)columns, (uint32_t)columns);
    }
    for (int i = p.copies; i < 4; ++i) p.pad.first[i + 1] = p.pad.first[p.copies];
    if (p.copies && features % 8) a.features = p.pad.padded;  // (then every matrix is a copy)
  }
  a.sums = (float*)((char*)workspace + p.bytes);
  p.bytes += sums_bytes(a, p.choice.splits);
  return HB_OK;
}

template <bool F16>
int launch(Plan& p, int count, hipStream_t st) {
  if (p.copies) {
    hipLaunchKernelGGL(pad_rows_kernel, dim3(std::min(p.pad.first[p.copies], PAD_GROUPS)), dim3(256), 0, st, p.pad);
    HB_HIP(hipGetLastError());
  }
  if (p.choice.kernel != FEW16) return launch_kernel<F16>(p.a, count, p.choice, st);
  p.a.tiles0 = (uint32_t)((p.a.columns + 15) / 16);
  hipLaunchKernelGGL((linear_few_kernel<F16>), dim3(p.a.tiles0 * count), dim3(64 * FEW_WAVES), 0, st, p.a);
  HB_HIP(hipGetLastError());
  return HB_OK;
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int64_t hb_linear_workspace_bytes(int32_t count, int32_t batch, const int32_t* rows, int32_t columns,
                                             int32_t features, void* const* pointers, const int64_t* strides) {
  Plan p;
  if (plan(p, count, batch, rows, columns, features, NONE, pointers, strides, nullptr)) return -1;
  const int64_t bytes = p.bytes;
  // (an activation before a residual only makes the wide kernel's whole sums slower, in favour of another kernel)
  if (p.choice.kernel != WIDE256 || p.choice.splits > 1 || !p.a.set[0].residual) return bytes;
  plan(p, count, batch, rows, columns, features, GELU, pointers, strides, nullptr);
  return std::max(bytes, p.bytes);
}

extern "C" int hb_linear_choice(int32_t count, int32_t batch, const int32_t* rows, int32_t columns, int32_t features,
                                int32_t act, void* const* pointers, const int64_t* strides, int32_t* choice) {
  HB_REQUIRE(choice, "null pointer argument");
  HB_REQUIRE(act >= 0 && act <= 2, "act must be 0 (none), 1 (GELU) or 2 (SiLU)");
  Plan p;
  const int rc = plan(p, count, batch, rows, columns, features, act, pointers, strides, nullptr);
  if (rc) return rc;
  const bool few = p.choice.kernel == FEW16, wide = p.choice.kernel == WIDE256 && p.choice.splits == 1;
  choice[0] = few ? 16 : SHAPES[p.choice.kernel].tc;
  choice[1] = few ? FEW_ROWS : SHAPES[p.choice.kernel].tt;
  choice[2] = p.choice.splits;
  choice[3] = wide && mode_of(p.a, count) == ANY;
  return HB_OK;
}

extern "C" int hb_linear(int32_t count, int32_t batch, const int32_t* rows, int32_t columns, int32_t features,
                         int32_t dtype, int32_t act, void* const* pointers, const int64_t* strides, void* workspace,
                         int64_t workspace_bytes, hb_stream_t stream) {
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16, "dtype must be bf16 or fp16");
  HB_REQUIRE(act >= 0 && act <= 2, "act must be 0 (none), 1 (GELU) or 2 (SiLU)");
  Plan p;
  const int rc = plan(p, count, batch, rows, columns, features, act, pointers, strides, workspace);
  if (rc) return rc;
  HB_REQUIRE(!p.bytes || (workspace && aligned16(workspace) && workspace_bytes >= p.bytes),
             "the workspace must hold %lld bytes, 16-byte aligned", (long long)p.bytes);
  return dtype == HB_DTYPE_F16 ? launch<true>(p, count, stream) : launch<false>(p, count, stream);
}
