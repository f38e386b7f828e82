// Group norm with an activation over images whose channels lie last in memory.
//
//   out = act((x - mean) / sqrt(var + eps) * weight + bias),  mean and var over a batch element's pixels and the
//   channels of a group;  act: none or SiLU
//
// The norm before every convolution of an image decoder.  HBM-bound: the values are read once for the statistics and once
// to be normalised, the second time from the caches where they fit.  Sums are fp32: a thread takes 8 pixels of 8 channels
// at a time, their means and centred squares exactly (two passes in registers), and joins those of different pixels and
// channels by their counts, means and squares (Chan's formula), so that a mean far from zero costs no precision.
//
//  * group_norm_few_kernel: a workgroup holds a group of an element in registers, one launch.
//  * group_norm_sums_kernel, group_norm_kernel: chunks of pixels by all channels; a chunk's means and squares per group
//    go through the workspace, and every workgroup of the second launch joins those of its element itself.  It walks
//    its chunk backwards: what the first launch read last is in the caches.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "../../include/hilberta_hip.h"

namespace hb {
namespace {

constexpr int V = 8;                  // channels of a thread
constexpr int THREADS = 256;
constexpr int MAX_CHANNELS = 8192;
constexpr int64_t CHUNK_BYTES = 64 << 10;
constexpr int MAX_CHUNKS = 512;       // of a launch

struct Args {
  const void* x;
  void* out;
  const void* weight;  // [channels] or null
  const void* bias;    // [channels] or null
  float2* sums;        // [batch, chunks, groups] mean and centred squares
  int64_t x_b, x_n, out_b, out_n;
  uint32_t pixels, chunk, chunks;  // of an element, of a chunk; chunks of an element
  int32_t channels, groups, per;   // per: channels of a group
  int32_t vectors, rows;           // threads along the channels, and along the pixels
  float eps;
  int32_t silu;
};

template <int DT>
struct Type {
  typedef uint16_t T;
};
template <>
struct Type<HB_DTYPE_F32> {
  typedef float T;
};

typedef u32x4 __attribute__((aligned(2))) words_at2;
typedef u32x4 __attribute__((aligned(4))) words_at4;
typedef f32x4 __attribute__((aligned(4))) floats_at4;

template <int DT>
__device__ __forceinline__ float value(const typename Type<DT>::T* p) {
  if constexpr (DT == HB_DTYPE_F32) return *p;
  else return to_f<DT == HB_DTYPE_F16>(*p);
}

// Eight values as they lie in memory.
template <int DT>
struct Raw {
  u32x4 v[DT == HB_DTYPE_F32 ? 2 : 1];
};
template <int DT, bool EDGE, bool STREAM>
__device__ __forceinline__ Raw<DT> load(const typename Type<DT>::T* p, int there) {
  Raw<DT> r = {};
  if (EDGE && there < V) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (k >= there) continue;
      if constexpr (DT == HB_DTYPE_F32) r.v[k >> 2][k & 3] = __builtin_bit_cast(uint32_t, p[k]);
      else r.v[0][k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
    }
    return r;
  }
  if constexpr (DT == HB_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) r.v[i] = STREAM ? __builtin_nontemporal_load((const words_at4*)(p + 4 * i)) : *(const words_at4*)(p + 4 * i);
  } else {
    r.v[0] = STREAM ? __builtin_nontemporal_load((const words_at2*)p) : *(const words_at2*)p;
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void unpack(const Raw<DT>& r, float (&x)[V]) {
  if constexpr (DT == HB_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // (whole vectors: of an element the builtin takes the first)
      const f32x4 v = __builtin_bit_cast(f32x4, r.v[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[4 * i + k] = v[k];
    }
  } else {
    unpack8<DT == HB_DTYPE_F16>(r.v[0], x);
  }
}
template <int DT, bool EDGE, bool STREAM>
__device__ __forceinline__ void store(typename Type<DT>::T* p, const float (&x)[V], int there) {
  if (EDGE && there < V) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (k >= there) continue;
      if constexpr (DT == HB_DTYPE_F32) p[k] = x[k];
      else p[k] = from_f<DT == HB_DTYPE_F16>(x[k]);
    }
    return;
  }
  if constexpr (DT == HB_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 v = {x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
      if constexpr (STREAM) __builtin_nontemporal_store(v, (floats_at4*)(p + 4 * i));
      else *(floats_at4*)(p + 4 * i) = v;
    }
  } else {
    const u32x4 v = pack8<DT == HB_DTYPE_F16>(x);
    if constexpr (STREAM) __builtin_nontemporal_store(v, (words_at2*)p);
    else *(words_at2*)p = v;
  }
}

__device__ __forceinline__ float activate(float v, int silu) {
  return silu ? v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)) : v;
}

// Mean and centred squares of n values.
struct Sums {
  float n, mean, squares;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float n = a.n + b.n, d = b.mean - a.mean, share = n > 0.f ? b.n * __builtin_amdgcn_rcpf(n) : 0.f;
  return {n, a.mean + d * share, a.squares + b.squares + d * d * a.n * share};
}

// ------------------------------------------------------------------ statistics of a chunk
template <int DT, bool EDGE>
__global__ void group_norm_sums_kernel(Args a) {
  typedef typename Type<DT>::T T;
  extern __shared__ float lds[];  // [2][rows][vectors * V]
  const int width = a.vectors * V, tx = threadIdx.x % a.vectors, ty = threadIdx.x / a.vectors;
  const uint32_t p0 = blockIdx.x * a.chunk, p1 = min(a.pixels, p0 + a.chunk), rows = a.rows;
  const int there = a.channels - tx * V;
  const T* const x = (const T*)a.x + blockIdx.y * a.x_b + tx * V;
  float mean[V] = {}, squares[V] = {}, n = 0.f;
  auto take = [&](uint32_t p, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    Raw<DT> raw[8];
    int count = 8;
    if (!WHOLE) count = (int)((p1 - p + rows - 1) / rows);
#pragma unroll
    for (int r = 0; r < 8; ++r) raw[r] = load<DT, EDGE, false>(x + (int64_t)(p + (WHOLE || r < count ? r : 0) * rows) * a.x_n, there);
    float v[8][V];
#pragma unroll
    for (int r = 0; r < 8; ++r) unpack(raw[r], v[r]);
    const float m = (float)count, inverse = WHOLE ? 0.125f : 1.f / m;
    const float share = m / (n + m), weight = n * share;
    n += m;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float sum = 0.f, square = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) sum += WHOLE || r < count ? v[r][k] : 0.f;
      const float center = sum * inverse;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float d = v[r][k] - center;
        square += WHOLE || r < count ? d * d : 0.f;
      }
      const float d = center - mean[k];
      mean[k] += d * share;
      squares[k] += square + d * d * weight;
    }
  };
  uint32_t p = p0 + ty;
  for (; p + 7 * rows < p1; p += 8 * rows) take(p, std::true_type());
  if (p < p1) take(p, std::false_type());
#pragma unroll
  for (int k = 0; k < V; ++k) {
    lds[ty * width + tx * V + k] = mean[k];
    lds[(rows + ty) * width + tx * V + k] = squares[k];
  }
  __syncthreads();
  // Eight lanes a group: its mean, then the squares about it.
  const int lanes = blockDim.x / 8, lane = threadIdx.x & 7, taken = p1 - p0;
  for (int g = threadIdx.x / 8; g < a.groups && (int)threadIdx.x < lanes * 8; g += lanes) {
    float sum = 0.f;
    for (uint32_t r = 0; r < rows; ++r) {
      const float count = (float)((taken - (int)r + (int)rows - 1) / (int)rows);
      for (int c = lane; c < a.per; c += 8) sum += count * lds[r * width + g * a.per + c];
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) sum += __shfl_xor(sum, m, 64);
    const float center = sum / ((float)taken * (float)a.per);
    float square = 0.f;
    for (uint32_t r = 0; r < rows; ++r) {
      const float count = (float)((taken - (int)r + (int)rows - 1) / (int)rows);
      for (int c = lane; c < a.per; c += 8) {
        const float d = lds[r * width + g * a.per + c] - center;
        square += lds[(rows + r) * width + g * a.per + c] + count * d * d;
      }
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) square += __shfl_xor(square, m, 64);
    if (lane == 0) a.sums[((int64_t)blockIdx.y * a.chunks + blockIdx.x) * a.groups + g] = {center, square};
  }
}

// ------------------------------------------------------------------ the values of a chunk
template <int DT, bool EDGE, bool STREAM>
__global__ void group_norm_kernel(Args a) {
  typedef typename Type<DT>::T T;
  extern __shared__ float lds[];  // [2][groups] mean and 1 / deviation
  const int tx = threadIdx.x % a.vectors, ty = threadIdx.x / a.vectors;
  int lanes = 64;  // that share a group
  while (lanes > 1 && lanes * a.groups > (int)blockDim.x) lanes >>= 1;
  const int together = blockDim.x / lanes, lane = threadIdx.x & (lanes - 1);
  const float2* const sums = a.sums + (int64_t)blockIdx.y * a.chunks * a.groups;
  for (int g = threadIdx.x / lanes; g < a.groups && (int)threadIdx.x < together * lanes; g += together) {
    Sums all = {0.f, 0.f, 0.f};
    for (uint32_t c = lane; c < a.chunks; c += lanes) {
      const float2 s = sums[(int64_t)c * a.groups + g];
      all = join(all, {(float)(min(a.pixels, (c + 1) * a.chunk) - c * a.chunk) * (float)a.per, s.x, s.y});
    }
    for (int m = 1; m < lanes; m <<= 1)
      all = join(all, {__shfl_xor(all.n, m, 64), __shfl_xor(all.mean, m, 64), __shfl_xor(all.squares, m, 64)});
    if (lane == 0) {
      lds[g] = all.mean;
      lds[a.groups + g] = __builtin_amdgcn_rsqf(all.squares / all.n + a.eps);
    }
  }
  __syncthreads();
  const int c0 = tx * V, there = a.channels - c0;
  float mean[V], scale[V], shift[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = min(c0 + k, a.channels - 1), g = c / a.per;
    mean[k] = lds[g];
    scale[k] = lds[a.groups + g] * (a.weight ? value<DT>((const T*)a.weight + c) : 1.f);
    shift[k] = a.bias ? value<DT>((const T*)a.bias + c) : 0.f;
  }
  const T* const x = (const T*)a.x + blockIdx.y * a.x_b + c0;
  T* const out = (T*)a.out + blockIdx.y * a.out_b + c0;
  const uint32_t p0 = blockIdx.x * a.chunk, p1 = min(a.pixels, p0 + a.chunk), rows = a.rows;
  constexpr int AT_ONCE = 4;
  // (backwards: the thread's last pixels first)
  for (int i = ((int)(p1 - p0) - ty + (int)rows - 1) / (int)rows - 1; i >= 0; i -= AT_ONCE) {
    Raw<DT> raw[AT_ONCE];
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) raw[r] = load<DT, EDGE, STREAM>(x + (int64_t)(p0 + ty + max(i - r, 0) * rows) * a.x_n, there);
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {
      if (i < r) break;
      float v[V];
      unpack(raw[r], v);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = activate((v[k] - mean[k]) * scale[k] + shift[k], a.silu);
      store<DT, EDGE, STREAM>(out + (int64_t)(p0 + ty + (i - r) * rows) * a.out_n, v, there);
    }
  }
}

// ------------------------------------------------------------------ groups that fit a workgroup
// W channels a load, up to UNITS loads a thread.
constexpr int UNITS = 8, FEW_THREADS = 1024;

template <int DT, int W>
__global__ __launch_bounds__(FEW_THREADS) void group_norm_few_kernel(Args a) {
  typedef typename Type<DT>::T T;
  __shared__ float parts[2][FEW_THREADS / 64];
  const int g = blockIdx.x, wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
  const uint32_t across = a.per / W, all = a.pixels * across;  // loads of a pixel, and of the group
  const T* const x = (const T*)a.x + blockIdx.y * a.x_b + g * a.per;
  T* const out = (T*)a.out + blockIdx.y * a.out_b + g * a.per;
  typedef T Unit __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  float v[UNITS][W];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const uint32_t at = i * blockDim.x + threadIdx.x, p = at / across, c = (at - p * across) * W;
    Unit u = {};
    if (at < all) u = *(const Unit*)(x + (int64_t)p * a.x_n + c);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if constexpr (DT == HB_DTYPE_F32) v[i][k] = u[k];
      else v[i][k] = to_f<DT == HB_DTYPE_F16>(u[k]);
      sum += v[i][k];  // (zeros past the group's values)
    }
  }
  auto total = [&](float s, float (&part)[FEW_THREADS / 64]) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    if ((threadIdx.x & 63) == 0) part[wave] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < waves; ++w) s += part[w];
    return s;
  };
  const float n = (float)all * W, mean = total(sum, parts[0]) / n;
  float squares = 0.f;
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
    if (i * blockDim.x + threadIdx.x < all) {
#pragma unroll
      for (int k = 0; k < W; ++k) squares += (v[i][k] - mean) * (v[i][k] - mean);
    }
  const float scale = __builtin_amdgcn_rsqf(total(squares, parts[1]) / n + a.eps);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const uint32_t at = i * blockDim.x + threadIdx.x, p = at / across, c = (at - p * across) * W;
    if (at >= all) break;
    Unit u;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float w = a.weight ? value<DT>((const T*)a.weight + g * a.per + c + k) : 1.f;
      const float b = a.bias ? value<DT>((const T*)a.bias + g * a.per + c + k) : 0.f;
      const float y = activate((v[i][k] - mean) * (scale * w) + b, a.silu);
      if constexpr (DT == HB_DTYPE_F32) u[k] = y;
      else u[k] = from_f<DT == HB_DTYPE_F16>(y);
    }
    *(Unit*)(out + (int64_t)p * a.out_n + c) = u;
  }
}

// ------------------------------------------------------------------ launches
int64_t size_of(int dtype) { return dtype == HB_DTYPE_F32 ? 4 : 2; }

// Channels of a load of group_norm_few_kernel: the most that divide a group's.
int few_width(int per) { return per % 8 == 0 ? 8 : per % 4 == 0 ? 4 : per % 2 == 0 ? 2 : 1; }

// Whether a workgroup holds a group (and the launch all of them: a grid holds fewer than 2^32 threads).
bool few(int64_t batch, int64_t pixels, int groups, int per) {
  return pixels * (per / few_width(per)) <= (int64_t)UNITS * FEW_THREADS / 4 && batch * groups < (1ll << 32) / FEW_THREADS;
}

struct Chunks {
  int64_t pixels, count;
};
Chunks chunks_of(int64_t batch, int64_t pixels, int channels, int dtype) {
  const int64_t row = channels * size_of(dtype), most = std::max<int64_t>(1, MAX_CHUNKS / batch);
  const int64_t count = std::clamp<int64_t>(pixels * row / CHUNK_BYTES, 1, most), each = (pixels + count - 1) / count;
  return {each, (pixels + each - 1) / each};
}

template <int DT, int W>
int launch_few(const Args& a, int32_t batch, hipStream_t st) {
  const int64_t units = (int64_t)a.pixels * (a.per / W);
  const int threads = (int)std::clamp<int64_t>((units + 63) / 64 * 64, 64, FEW_THREADS);
  hipLaunchKernelGGL((group_norm_few_kernel<DT, W>), dim3(a.groups, batch), dim3(threads), 0, st, a);
  HB_HIP(hipGetLastError());
  return HB_OK;
}

template <int DT, bool EDGE>
int launch_chunks(const Args& a, int32_t batch, bool stream_values, hipStream_t st) {
  const dim3 grid(a.chunks, batch), block(a.vectors * a.rows);
  hipLaunchKernelGGL((group_norm_sums_kernel<DT, EDGE>), grid, block, block.x * V * 2 * sizeof(float), st, a);
  HB_HIP(hipGetLastError());
  const size_t lds = 2 * a.groups * sizeof(float);
  if (stream_values) hipLaunchKernelGGL((group_norm_kernel<DT, EDGE, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((group_norm_kernel<DT, EDGE, false>), grid, block, lds, st, a);
  HB_HIP(hipGetLastError());
  return HB_OK;
}

template <int DT>
int launch(Args& a, int32_t batch, hipStream_t st) {
  if (few(batch, a.pixels, a.groups, a.per)) {
    switch (few_width(a.per)) {
      case 8: return launch_few<DT, 8>(a, batch, st);
      case 4: return launch_few<DT, 4>(a, batch, st);
      case 2: return launch_few<DT, 2>(a, batch, st);
      default: return launch_few<DT, 1>(a, batch, st);
    }
  }
  const bool stream_values = 2 * (int64_t)batch * a.pixels * a.channels * size_of(DT) > CACHE_BYTES;
  return a.channels % V ? launch_chunks<DT, true>(a, batch, stream_values, st) : launch_chunks<DT, false>(a, batch, stream_values, st);
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int64_t hb_group_norm_workspace_bytes(int32_t batch, int64_t pixels, int32_t channels, int32_t groups, int32_t dtype) {
  if (batch < 1 || pixels < 1 || channels < 1 || groups < 1 || channels % groups || dtype < 0 || dtype > HB_DTYPE_F32) return -1;
  if (few(batch, pixels, groups, channels / groups)) return 0;
  return batch * chunks_of(batch, pixels, channels, dtype).count * groups * (int64_t)sizeof(float2);
}

extern "C" int hb_group_norm(int32_t batch, int64_t pixels, int32_t channels, int32_t groups, int32_t dtype, int32_t silu,
                             float eps, const void* x, int64_t x_batch_stride, int64_t x_pixel_stride, const void* weight,
                             const void* bias, void* out, int64_t out_batch_stride, int64_t out_pixel_stride,
                             void* workspace, int64_t workspace_bytes, hb_stream_t stream) {
  HB_REQUIRE(x && out, "null pointer argument");
  HB_REQUIRE(batch > 0 && batch <= 65535 && pixels > 0 && pixels < (1ll << 31), "batch must be in [1, 65535] and pixels in [1, 2^31)");
  HB_REQUIRE(channels > 0 && channels <= MAX_CHANNELS, "channels must be in [1, %d] (got %d)", MAX_CHANNELS, channels);
  HB_REQUIRE(groups > 0 && channels % groups == 0, "groups must divide the channels");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16 || dtype == HB_DTYPE_F32, "dtype must be bf16, fp16 or fp32");
  HB_REQUIRE(silu == 0 || silu == 1, "silu must be 0 or 1");
  HB_REQUIRE(eps > 0.f, "eps must be positive");
  const uintptr_t size = (uintptr_t)size_of(dtype);
  HB_REQUIRE((((uintptr_t)x | (uintptr_t)weight | (uintptr_t)bias | (uintptr_t)out) & (size - 1)) == 0, "every pointer must be aligned to its elements");
  HB_REQUIRE(x_batch_stride >= 0 && x_pixel_stride >= 0 && out_batch_stride >= 0 && out_pixel_stride >= 0, "strides must be non-negative");
  Args a = {};
  a.x = x;
  a.out = out;
  a.weight = weight;
  a.bias = bias;
  a.x_b = x_batch_stride;
  a.x_n = x_pixel_stride;
  a.out_b = out_batch_stride;
  a.out_n = out_pixel_stride;
  a.pixels = (uint32_t)pixels;
  a.channels = channels;
  a.groups = groups;
  a.per = channels / groups;
  a.eps = eps;
  a.silu = silu;
  a.vectors = (channels + V - 1) / V;
  a.rows = std::max(1, THREADS / a.vectors);
  const int64_t need = hb_group_norm_workspace_bytes(batch, pixels, channels, groups, dtype);
  if (need) {
    HB_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need, "the workspace must hold %lld bytes, 8-byte aligned", (long long)need);
    const Chunks c = chunks_of(batch, pixels, channels, dtype);
    a.sums = (float2*)workspace;
    a.chunk = (uint32_t)c.pixels;
    a.chunks = (uint32_t)c.count;
  }
  switch (dtype) {
    case HB_DTYPE_BF16: return launch<HB_DTYPE_BF16>(a, batch, stream);
    case HB_DTYPE_F16: return launch<HB_DTYPE_F16>(a, batch, stream);
    default: return launch<HB_DTYPE_F32>(a, batch, stream);
  }
}
