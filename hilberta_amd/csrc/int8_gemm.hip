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
// columns: a lane then holds one token's values, 4 consecutive channels an accumulator quarter, so that a
// token's scale is one register, a rotated pair lies in one lane, and a head's 128 channels in the lanes l
// and l + 32.
#include "common.h"
#include "../../include/hilberta_hip.h"

namespace hb {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int MAX_FEATURES = 1 << 17;
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
  // v (1 + tanh u) / 2 = v / (1 + exp(-2u)),  u = sqrt(2 / pi) (v + 0.044715 v^3)
  const float u = v * (0.7978845608028654f + 0.035677408136300125f * v * v);
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-2.885390081777927f * u));
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

// s_waitcnt vmcnt(N) lgkmcnt(0)
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

constexpr int TC = 128, TT = 256;              // channels and tokens of a workgroup's tile
constexpr int STEP = 64;                       // features of a stage: bytes of an LDS row
constexpr int STAGE = (TC + TT) * STEP;        // 24 KB
constexpr int LOADS = STAGE / 1024 / 4;        // 1 KB loads of a wave and stage
constexpr int BAND = 8;                        // token tiles walked together

template <bool F16, bool QKV, bool GELU>
__global__ __launch_bounds__(256, 2) void int8_product_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) int8_t lds0[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds1[STAGE];
  __shared__ __attribute__((aligned(1024))) int8_t lds2[STAGE];
  __shared__ __attribute__((aligned(16))) float channel[3][TC];  // weight scale, bias, head norm
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  // Workgroups go to the eight XCDs in turn: each XCD takes a run of tiles, in bands of BAND token tiles
  // walked channel tile by channel tile, so that its L2 serves a patch of both operands.
  uint32_t tile = (blockIdx.x & 7) * a.tiles_xcd + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= a.tiles_xcd || tile >= a.tiles) return;
  const bool second = tile >= a.tiles0;
  const Set& s = a.set[second];
  if (second) tile -= a.tiles0;
  const uint32_t token_tiles = (s.tokens + TT - 1) / TT;
  const uint32_t band = tile / (BAND * a.channel_tiles), in_band = tile - band * (BAND * a.channel_tiles);
  const uint32_t height = min((uint32_t)BAND, token_tiles - band * BAND);
  const uint32_t ct = in_band / height;
  const int c0 = ct * TC;
  const uint32_t t0 = (band * BAND + in_band - ct * height) * TT;
  const int plane = QKV ? c0 / (a.heads * HEAD) : 2;
  for (int i = threadIdx.x; i < TC; i += 256) {
    const int c = min(c0 + i, a.columns - 1);
    channel[0][i] = s.w_scale[c];
    channel[1][i] = s.bias ? to_f<F16>(s.bias[c]) : 0.f;
    channel[2][i] = QKV && plane < 2 && s.norm[plane] ? to_f<F16>(s.norm[plane][i]) : 1.f;
  }
  // Loads: a wave's load j fills LDS rows 16 (4 j + wave) .. + 15, four lanes a row of 64 bytes; rows below
  // TC are channels, the others tokens.  The lane at slot p of row r loads chunk p ^ (r / 4 % 4), so that
  // the 16 rows whose chunks a quarter of a wave reads together lie in different banks.
  const int8_t* wbase = s.w + (int64_t)c0 * a.padded;
  const int8_t* qbase = s.q + (int64_t)t0 * a.padded;
  int offset[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = 16 * (4 * j + wave) + (lane >> 2);
    const int chunk = (lane & 3) ^ (r >> 2 & 3);
    const int row = 4 * j < TC / 16 ? min(r, a.columns - 1 - c0) : (int)min((uint32_t)(r - TC), s.tokens - 1 - t0);
    offset[j] = row * a.padded + chunk * 16;
  }
  const int stages = a.padded / STEP;
  auto load = [&](int8_t* dst, int stage) {
    const int at = min(stage, stages - 1) * STEP;  // (past the end: the last stage again, never read)
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      load_lds16(4 * j < TC / 16 ? wbase : qbase, dst + 1024 * (4 * j + wave), offset[j], at);
  };
  // Operands: lane l holds bytes 16 (l / 32) .. + 15 of a 32-byte step of row l % 32.
  const int swizzle = (col >> 2 & 3) ^ half;
  const int read = col * STEP + swizzle * 16;
  i32x4 w[2][4], x[2][2];
  auto fetch = [&](const int8_t* src, int u) {
    const int at = read ^ (u * 32);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[u][i] = *(const i32x4*)(src + i * 32 * STEP + at);
#pragma unroll
    for (int j = 0; j < 2; ++j) x[u][j] = *(const i32x4*)(src + (TC + wave * 64 + j * 32) * STEP + at);
  };
  i32x16 acc[4][2] = {};
  auto multiply = [&](int u) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[u][i], x[u][j], acc[i][j], 0, 0, 0);
  };
  // Stage n is in `cur`, its first operands in w[0], x[0]; stage n + 1 is on its way to `next`.  The barrier
  // says that everyone's part of it is there, and that nobody still reads `cur`, which stage n + 3 will fill.
  auto step = [&](int8_t* cur, int8_t* next, int8_t* last, int n) {
    load(last, n + 2);
    fetch(cur, 1);
    multiply(0);
    wait_loads<LOADS>();
    barrier();
    fetch(next, 0);
    multiply(1);
  };
  load(lds0, 0);
  load(lds1, 1);
  wait_loads<LOADS>();
  __syncthreads();
  fetch(lds0, 0);
  for (int n = 0;;) {
    step(lds0, lds1, lds2, n);
    if (++n == stages) break;
    step(lds1, lds2, lds0, n);
    if (++n == stages) break;
    step(lds2, lds0, lds1, n);
    if (++n == stages) break;
  }
  wait_loads<0>();  // (nothing may still be on its way to LDS when the workgroup ends)
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t at = t0 + wave * 64 + j * 32 + col, token = min(at, s.tokens - 1);
    const float scale = s.scale[token];
    const uint32_t b = token / s.rows, n = token - b * s.rows;
    uint16_t* out = s.out + b * s.out_b + (int64_t)n * s.out_n;
    const float *co = nullptr, *si = nullptr;
    float v[4][16];
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = i * 32 + g * 8 + half * 4;
        const f32x4 ws = *(const f32x4*)&channel[0][c], bias = *(const f32x4*)&channel[1][c];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float p = (float)acc[i][j][g * 4 + k] * scale * ws[k] + bias[k];
          if (QKV) squares += p * p;
          if (GELU) p = gelu(p);
          v[i][g * 4 + k] = p;
        }
      }
    if (QKV) {
      out += plane * a.out_p + (c0 - plane * a.heads * HEAD);
      if (plane < 2) {
        squares += __shfl_xor(squares, 32, 64);
        const float rms = __builtin_amdgcn_rsqf(squares * (1.f / HEAD) + a.eps);
        co = a.cos ? a.cos + (int64_t)(s.first + n) * HEAD : nullptr;
        si = a.cos ? a.sin + (int64_t)(s.first + n) * HEAD : nullptr;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int c = i * 32 + g * 8 + half * 4;
            const f32x4 norm = *(const f32x4*)&channel[2][c];
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = v[i][g * 4 + k] * rms * norm[k];
            if (a.cos) {
              const f32x4 cv = *(const f32x4*)(co + c), sv = *(const f32x4*)(si + c);
#pragma unroll
              for (int k = 0; k < 4; k += 2) {
                v[i][g * 4 + k] = y[k] * cv[k] - y[k + 1] * sv[k];
                v[i][g * 4 + k + 1] = y[k + 1] * cv[k + 1] + y[k] * sv[k + 1];
              }
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) v[i][g * 4 + k] = y[k];
            }
          }
      }
    } else {
      out += c0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float even[4], odd[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          even[k] = v[i][8 * p + k];
          odd[k] = v[i][8 * p + 4 + k];
        }
        const u32x4 packed = pack_pair<F16>(even, odd);
        const int c = i * 32 + p * 16 + half * 8;
        if (at < s.tokens) {
          if (QKV || (a.vectors && c0 + c + 8 <= a.columns)) {
            *(u32x4*)(out + c) = packed;
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (c0 + c + k < a.columns) out[c + k] = (uint16_t)(packed[k >> 1] >> (16 * (k & 1)));
          }
        }
      }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <bool F16, bool QKV>
void launch_type(const Args& a, hipStream_t st) {
  const dim3 grid(8 * a.tiles_xcd), block(256);
  if (a.gelu) hipLaunchKernelGGL((int8_product_kernel<F16, QKV, !QKV>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((int8_product_kernel<F16, QKV, false>), grid, block, 0, st, a);
}

template <bool QKV>
int launch(Args& a, int count, int32_t dtype, hipStream_t st) {
  a.channel_tiles = (uint32_t)((a.columns + TC - 1) / TC);
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) {
    tiles += (int64_t)((a.set[i].tokens + TT - 1) / TT) * a.channel_tiles;
    HB_REQUIRE(tiles < (1ll << 30), "too many output tiles for one launch");
    if (i == 0) a.tiles0 = (uint32_t)tiles;
  }
  a.tiles = (uint32_t)tiles;
  a.tiles_xcd = (a.tiles + 7) / 8;
  if (dtype == HB_DTYPE_F16) launch_type<true, QKV>(a, st);
  else launch_type<false, QKV>(a, st);
  HB_HIP(hipGetLastError());
  return HB_OK;
}

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
         (uint16_t*)p[5], {nullptr, nullptr}, strides[2 * i], strides[2 * i + 1], (uint32_t)rows[i], 0, 0};
    const int rc = check_set(s, batch, rows[i], padded);
    if (rc) return rc;
    s.tokens = (uint32_t)(batch * rows[i]);
    a.vectors &= aligned16(s.out) && s.out_b % 8 == 0 && s.out_n % 8 == 0;
  }
  return launch<false>(a, count, dtype, stream);
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
         out_row_stride, (uint32_t)rows, 0, (uint32_t)first};
    const int rc = check_set(s, batch, rows, padded);
    if (rc) return rc;
    HB_REQUIRE(((uintptr_t)s.norm[0] & 1) == 0 && ((uintptr_t)s.norm[1] & 1) == 0, "norm weights must be 2-byte aligned");
    s.tokens = (uint32_t)(batch * rows);
  }
  return launch<true>(a, count, dtype, stream);
}
