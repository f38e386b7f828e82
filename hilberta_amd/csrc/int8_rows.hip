// 16-bit rows to 8-bit rows with one scale a row, alone and as the end of the gated residual + AdaLN pass.
//
// For a row x of `features` values, all in fp32:
//   top = max |x_k|,  scale = top / 127,  q_k = rint(127 x_k / top)  (ties to even; a row of zeros: all zero)
// A row that holds an infinity or a NaN gets the scale NaN (and q = 0), so that every product with it is
// NaN.  q rows are filled up with zeros to `padded` columns, a multiple of 64, which the product walks whole.
//
// (q is exact: int8_common.h.)
#include "int8_common.h"
#include "../../include/hilberta_hip.h"

namespace hb {
namespace {

constexpr uint32_t GRID_BLOCKS = (1 << 24) - 1;  // of 256 threads (a grid holds fewer than 2^32)
constexpr int WAVE_FEATURES = 3072;        // a row up to here is a wave's, a longer one a workgroup's

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m, 64));
  return v;
}

struct RowArgs {
  const uint16_t* x;
  int64_t x_b, x_n;  // batch and row strides
  int8_t* q;         // [rows of all batches, padded]
  float* scale;
  uint32_t rows, total;  // of a batch element, and of all
  int32_t features, padded;
};

// LANES (a wave or a workgroup of 256) hold a row, NV vectors of 8 values each, and read it once; a row longer
// than that (NV = 0) is read again for its whole numbers.  Bound by memory: 16384 x 12288 (604 MB) 90 us, 6.7
// TB/s, read past the caches (141 when every row was read twice), 16384 x 3072 (151 MB) 25 us, 6.0 TB/s.
template <bool F16, int LANES, int NV, bool STREAM>
__global__ __launch_bounds__(256) void int8_rows_kernel(RowArgs a) {
  __shared__ uint32_t tops[4];
  const uint32_t lane = threadIdx.x % LANES, row = blockIdx.x * (256u / LANES) + threadIdx.x / LANES;
  if (LANES == 64 && row >= a.total) return;  // the whole wave leaves together
  const uint32_t b = row / a.rows, i = row - b * a.rows;
  const uint16_t* x = a.x + b * a.x_b + (int64_t)i * a.x_n;
  int8_t* q = a.q + (int64_t)row * a.padded;
  u32x4 raw[NV ? NV : 1];
  u16x2 pairs = {0, 0};
  if constexpr (NV) {
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = load_row8<STREAM>(x, (v * LANES + lane) * 8, a.features);
#pragma unroll
    for (int v = 0; v < NV; ++v) pairs = max_pairs(pairs, raw[v]);
  } else {
    for (int col = lane * 8; col < a.features; col += LANES * 8) pairs = max_pairs(pairs, load_row8<false>(x, col, a.features));
  }
  uint32_t top = wave_max(fp32_bits<F16>(pairs));
  if constexpr (LANES == 256) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  const Scaler s(top);
  if constexpr (NV) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * LANES + lane) * 8;
      float values[8];
      unpack8<F16>(raw[v], values);
      if (col < a.padded) *(u32x2*)(q + col) = pack_row8(s, values);
    }
  } else {
    for (int col = lane * 8; col < a.padded; col += LANES * 8) {
      float values[8];
      unpack8<F16>(load_row8<false>(x, col, a.features), values);
      *(u32x2*)(q + col) = pack_row8(s, values);
    }
  }
  if (lane == 0) a.scale[row] = s.scale;
}

template <bool F16, bool STREAM>
void launch_rows(const RowArgs& a, hipStream_t st) {
  const dim3 waves((a.total + 3) / 4), groups(a.total), block(256);
  const int nv = (a.padded + 511) / 512;
  if (nv <= 1) hipLaunchKernelGGL((int8_rows_kernel<F16, 64, 1, STREAM>), waves, block, 0, st, a);
  else if (nv <= 2) hipLaunchKernelGGL((int8_rows_kernel<F16, 64, 2, STREAM>), waves, block, 0, st, a);
  else if (nv <= 4) hipLaunchKernelGGL((int8_rows_kernel<F16, 64, 4, STREAM>), waves, block, 0, st, a);
  else if (nv <= 6) hipLaunchKernelGGL((int8_rows_kernel<F16, 64, 6, STREAM>), waves, block, 0, st, a);
  else if (nv <= 8) hipLaunchKernelGGL((int8_rows_kernel<F16, 256, 2, STREAM>), groups, block, 0, st, a);
  else if (nv <= 16) hipLaunchKernelGGL((int8_rows_kernel<F16, 256, 4, STREAM>), groups, block, 0, st, a);
  else if (nv <= 24) hipLaunchKernelGGL((int8_rows_kernel<F16, 256, 6, STREAM>), groups, block, 0, st, a);
  else if (nv <= 32) hipLaunchKernelGGL((int8_rows_kernel<F16, 256, 8, STREAM>), groups, block, 0, st, a);
  else hipLaunchKernelGGL((int8_rows_kernel<F16, 256, 0, false>), groups, block, 0, st, a);
}

struct AdaRows {
  const uint16_t *x, *y, *gate;  // y null: no residual
  uint16_t* x_out;               // null: the residual is not stored
  const uint16_t *shift, *factor;
  int8_t* q;
  float* scale;
  int64_t x_b, x_n, y_b, y_n, gate_b, xo_b, xo_n, mod_b;
  uint32_t rows;
};

// Two row sets of one shape share a launch; the first `rows0` of `total` rows are a[0]'s.
struct AdaSets {
  AdaRows a[2];
  uint32_t rows0, total;
  int32_t hidden, padded;
  float inv_hidden, eps;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// r = x + gate y;  m = shift + LayerNorm(r) (1 + factor), in fp32, and m to 8 bits.  One wave a row, which
// it holds in registers: NV vectors of 8 values a lane.  The residual is stored rounded, and normalised
// before that rounding.  Bound by memory: 16384 x 3072 with a residual (353 MB) 69 us, 5.1 TB/s, without one (151 MB)
// 36 us.
template <bool F16, int NV, bool STREAM>
__global__ __launch_bounds__(256) void int8_adaln_kernel(AdaSets p) {
  uint32_t row = blockIdx.x * 4u + (threadIdx.x >> 6);
  if (row >= p.total) return;  // the whole wave leaves together
  const bool second = (uint32_t)uniform(row) >= p.rows0;
  const AdaRows& a = p.a[second];
  if (second) row -= p.rows0;
  const uint32_t lane = threadIdx.x & 63, b = row / a.rows, i = row - b * a.rows;
  const uint16_t* x = a.x + b * a.x_b + (int64_t)i * a.x_n;
  float r[NV][8];
  float sum = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = v * 512 + lane * 8;
    u32x4 raw = {0, 0, 0, 0};
    if (col < p.hidden) raw = load_once<STREAM>((const u32x4*)(x + col));
    unpack8<F16>(raw, r[v]);
  }
  if (a.y) {
    const uint16_t* y = a.y + b * a.y_b + (int64_t)i * a.y_n;
    const uint16_t* g = a.gate + b * a.gate_b;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = v * 512 + lane * 8;
      if (col < p.hidden) {
        float yv[8], gv[8];
        unpack8<F16>(load_once<STREAM>((const u32x4*)(y + col)), yv);
        unpack8<F16>(*(const u32x4*)(g + col), gv);
#pragma unroll
        for (int k = 0; k < 8; ++k) r[v][k] += gv[k] * yv[k];
        if (a.x_out) store_once<STREAM>((u32x4*)(a.x_out + b * a.xo_b + (int64_t)i * a.xo_n + col), pack8<F16>(r[v]));
      }
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += r[v][k];
  const float mean = wave_sum(sum) * p.inv_hidden;
  float sq = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const bool in = v * 512 + lane * 8 < p.hidden;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r[v][k] = in ? r[v][k] - mean : 0.f;
      sq += r[v][k] * r[v][k];
    }
  }
  const float rstd = __builtin_amdgcn_rsqf(wave_sum(sq) * p.inv_hidden + p.eps);
  uint32_t top = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = v * 512 + lane * 8;
    if (col < p.hidden) {
      float sh[8], sc[8];
      unpack8<F16>(*(const u32x4*)(a.shift + b * a.mod_b + col), sh);
      unpack8<F16>(*(const u32x4*)(a.factor + b * a.mod_b + col), sc);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        r[v][k] = sh[k] + r[v][k] * rstd * (1.f + sc[k]);
        top = max(top, __builtin_bit_cast(uint32_t, r[v][k]) & 0x7fffffffu);
      }
    }
  }
  const Scaler s(wave_max(top));
  int8_t* q = a.q + (int64_t)row * p.padded;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = v * 512 + lane * 8;
    if (col < p.padded) *(u32x2*)(q + col) = pack_row8(s, r[v]);
  }
  if (lane == 0) a.scale[row] = s.scale;
}

template <bool F16, bool STREAM>
void launch_adaln(const AdaSets& p, hipStream_t st) {
  const dim3 grid((p.total + 3) / 4), block(256);
  const int nv = (p.padded + 511) / 512;
  if (nv <= 1) hipLaunchKernelGGL((int8_adaln_kernel<F16, 1, STREAM>), grid, block, 0, st, p);
  else if (nv <= 2) hipLaunchKernelGGL((int8_adaln_kernel<F16, 2, STREAM>), grid, block, 0, st, p);
  else if (nv <= 4) hipLaunchKernelGGL((int8_adaln_kernel<F16, 4, STREAM>), grid, block, 0, st, p);
  else if (nv <= 6) hipLaunchKernelGGL((int8_adaln_kernel<F16, 6, STREAM>), grid, block, 0, st, p);
  else if (nv <= 8) hipLaunchKernelGGL((int8_adaln_kernel<F16, 8, STREAM>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((int8_adaln_kernel<F16, 16, STREAM>), grid, block, 0, st, p);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int hb_int8_rows(const void* x, int64_t batch_stride, int64_t row_stride, int32_t batch, int32_t rows,
                            int32_t features, int32_t padded, int32_t dtype, int8_t* q, float* scale,
                            hb_stream_t stream) {
  HB_REQUIRE(batch > 0 && rows > 0 && (int64_t)batch * rows < (1ll << 31), "batch and rows must be positive, with fewer than 2^31 rows in all");
  HB_REQUIRE(features > 0 && features <= MAX_FEATURES, "features must be in [1, %d] (got %d)", MAX_FEATURES, features);
  HB_REQUIRE(padded >= features && padded % 64 == 0 && padded <= MAX_FEATURES, "padded must be a multiple of 64, no smaller than features");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16, "dtype must be bf16 or fp16");
  HB_REQUIRE(x && q && scale, "null pointer argument");
  HB_REQUIRE(((uintptr_t)x & 1) == 0 && aligned16(q) && ((uintptr_t)scale & 3) == 0, "x must be 2-byte, q 16-byte and scale 4-byte aligned");
  HB_REQUIRE(batch_stride >= 0 && row_stride >= 0, "strides must be non-negative");
  const uint32_t total = (uint32_t)(batch * rows);
  HB_REQUIRE(total <= (padded <= WAVE_FEATURES ? GRID_BLOCKS * 4 : GRID_BLOCKS), "too many rows for one launch");
  const RowArgs a = {(const uint16_t*)x, batch_stride, row_stride, q, scale, (uint32_t)rows, total, features, padded};
  const bool repeats = (batch > 1 && batch_stride == 0) || (rows > 1 && row_stride == 0);
  const bool stream_in = (int64_t)total * features * 3 > CACHE_BYTES && !repeats;
  if (dtype == HB_DTYPE_F16) {
    if (stream_in) launch_rows<true, true>(a, stream);
    else launch_rows<true, false>(a, stream);
  } else {
    if (stream_in) launch_rows<false, true>(a, stream);
    else launch_rows<false, false>(a, stream);
  }
  HB_HIP(hipGetLastError());
  return HB_OK;
}

extern "C" int hb_int8_adaln(int32_t count, int32_t batch, const int32_t* rows, int32_t hidden, int32_t padded,
                             int32_t dtype, float eps, void* const* pointers, const int64_t* strides,
                             hb_stream_t stream) {
  HB_REQUIRE(count == 1 || count == 2, "count must be 1 or 2");
  HB_REQUIRE(rows && pointers && strides, "null pointer argument");
  HB_REQUIRE(hidden > 0 && hidden % 8 == 0 && hidden <= 8192, "hidden must be a multiple of 8 up to 8192 (got %d)", hidden);
  HB_REQUIRE(padded >= hidden && padded % 64 == 0 && padded <= 8192, "padded must be a multiple of 64, no smaller than hidden");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16, "dtype must be bf16 or fp16");
  HB_REQUIRE(eps > 0.f, "eps must be positive");
  AdaSets p = {};
  int64_t total = 0, bytes = 0;
  bool repeats = false;
  for (int i = 0; i < count; ++i) {
    void* const* q = pointers + 8 * i;
    const int64_t* s = strides + 8 * i;
    HB_REQUIRE(batch > 0 && rows[i] > 0, "batch and rows must be positive");
    total += (int64_t)batch * rows[i];
    HB_REQUIRE(total <= GRID_BLOCKS * 4, "too many rows for one launch");
    HB_REQUIRE(q[0] && q[4] && q[5] && q[6] && q[7], "null pointer argument");
    HB_REQUIRE((q[1] == nullptr) == (q[2] == nullptr), "y and gate are given together");
    HB_REQUIRE(!q[3] || q[1], "x_out is written only with a residual update");
    for (int k = 0; k < 7; ++k) HB_REQUIRE(aligned16(q[k]), "every pointer must be 16-byte aligned");
    HB_REQUIRE(((uintptr_t)q[7] & 3) == 0, "row scales must be 4-byte aligned");
    for (int k = 0; k < 8; ++k)
      HB_REQUIRE(s[k] >= 0 && s[k] % 8 == 0, "strides must be non-negative multiples of 8");
    bytes += (int64_t)batch * rows[i] * hidden * (2 * (1 + (q[1] != nullptr) + (q[3] != nullptr)) + 1);
    repeats |= (batch > 1 && (s[0] == 0 || (q[1] && s[2] == 0))) || (rows[i] > 1 && (s[1] == 0 || (q[1] && s[3] == 0)));
    p.a[i] = {(const uint16_t*)q[0], (const uint16_t*)q[1], (const uint16_t*)q[2], (uint16_t*)q[3],
              (const uint16_t*)q[4], (const uint16_t*)q[5], (int8_t*)q[6], (float*)q[7],
              s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], (uint32_t)rows[i]};
    if (i == 0) p.rows0 = (uint32_t)total;
  }
  p.total = (uint32_t)total;
  p.hidden = hidden;
  p.padded = padded;
  p.inv_hidden = 1.f / (float)hidden;
  p.eps = eps;
  const bool stream_in = bytes > CACHE_BYTES && !repeats;
  if (dtype == HB_DTYPE_F16) {
    if (stream_in) launch_adaln<true, true>(p, stream);
    else launch_adaln<true, false>(p, stream);
  } else {
    if (stream_in) launch_adaln<false, true>(p, stream);
    else launch_adaln<false, false>(p, stream);
  }
  HB_HIP(hipGetLastError());
  return HB_OK;
}
