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
constexpr int THREADS = 256, MAX_THREADS = 1024;
constexpr int MAX_CHANNELS = 8192;
constexpr int64_t CHUNK_BYTES = 16 << 10;
constexpr int64_t LARGE_BYTES = 512ll << 20, LARGE_FLOAT_BYTES = 640ll << 20;
constexpr int64_t LINE = 128;         // bytes of a cache line

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
// How rows divide into vectors: evenly; with a last vector that begins eight channels before the row's end and shares some
// with the one before; not at all, where there are fewer than eight channels (`there` of them).
enum Edge { EVEN, SHARED, SHORT };

template <int DT, int EDGE, bool STREAM>
__device__ __forceinline__ Raw<DT> load(const typename Type<DT>::T* p, int there) {
  Raw<DT> r = {};
  if (EDGE == SHORT) {
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
// (skip: the first channels that the vector before this one stores)
template <int DT, int EDGE, bool STREAM>
__device__ __forceinline__ void store(typename Type<DT>::T* p, const float (&x)[V], int skip, int there) {
  if (EDGE == SHORT || (EDGE == SHARED && skip)) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (k < skip || k >= there) continue;
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
template <int DT, int EDGE>
__global__ void group_norm_sums_kernel(Args a) {
  typedef typename Type<DT>::T T;
  extern __shared__ float lds[];  // [2][rows][vectors * V]
  const int width = a.vectors * V, tx = threadIdx.x % a.vectors, ty = threadIdx.x / a.vectors;
  const uint32_t p0 = blockIdx.x * a.chunk, p1 = min(a.pixels, p0 + a.chunk), rows = a.rows;
  const int first = EDGE == SHARED ? min(tx * V, a.channels - V) : tx * V, there = a.channels;
  const T* const x = (const T*)a.x + blockIdx.y * a.x_b + first;
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
    lds[ty * width + first + k] = mean[k];  // (channels that two vectors share: the same values twice)
    lds[(rows + ty) * width + first + k] = squares[k];
  }
  __syncthreads();
  // `lanes` neighbouring threads a group: its mean, then the squares about it.
  int lanes = 64;
  while (lanes > 1 && lanes * a.groups > (int)blockDim.x) lanes >>= 1;
  const int together = blockDim.x / lanes, lane = threadIdx.x & (lanes - 1), taken = p1 - p0, values = rows * a.per;
  // (the pixels of a row of threads: base, and one more of the first; where a lane begins, and its step)
  const int more = taken % (int)rows, r0 = lane / a.per, c0 = lane - r0 * a.per, dr = lanes / a.per, dc = lanes - dr * a.per;
  const float base = (float)(taken / (int)rows);
  for (int g = threadIdx.x / lanes; g < a.groups && (int)threadIdx.x < together * lanes; g += together) {
    auto sum_of = [&](auto term) {
      float sum = 0.f;
      int r = r0, c = c0;
#pragma unroll 4
      for (int e = lane; e < values; e += lanes) {
        sum += term(base + (r < more ? 1.f : 0.f), r * width + g * a.per + c);
        r += dr;
        c += dc;
        if (c >= a.per) c -= a.per, ++r;
      }
      for (int m = 1; m < lanes; m <<= 1) sum += __shfl_xor(sum, m, 64);
      return sum;
    };
    const float center = sum_of([&](float count, int at) { return count * lds[at]; }) / ((float)taken * (float)a.per);
    const float square = sum_of([&](float count, int at) {
      const float d = lds[at] - center;
      return lds[rows * width + at] + count * d * d;
    });
    if (lane == 0) a.sums[((int64_t)blockIdx.y * a.chunks + blockIdx.x) * a.groups + g] = {center, square};
  }
}

// ------------------------------------------------------------------ the values of a chunk
// The element's means and 1 / deviations of all groups: neighbouring threads take neighbouring groups, whose sums lie
// together, `lanes` threads a group its chunks in turn, eight loads at a time; what they have meets in LDS.
__device__ __forceinline__ void join_chunks(const Args& a, float* lds) {
  __shared__ Sums part[MAX_THREADS];
  int lanes = 1;
  while (2 * lanes * a.groups <= (int)blockDim.x && lanes < (int)a.chunks) lanes *= 2;
  const float2* const sums = a.sums + (int64_t)blockIdx.y * a.chunks * a.groups;
  const float each = (float)a.chunk * (float)a.per;
  for (int g0 = 0; g0 < a.groups; g0 += blockDim.x) {
    const int here = min(a.groups - g0, (int)blockDim.x), lane = threadIdx.x / here, g = g0 + threadIdx.x - lane * here;
    Sums all = {0.f, 0.f, 0.f};
    if (lane < lanes) {
      for (uint32_t c = lane; c < a.chunks; c += 8 * lanes) {
        float2 s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = sums[(int64_t)min(c + i * lanes, a.chunks - 1) * a.groups + g];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t at = c + i * lanes;
          const float n = at >= a.chunks ? 0.f : at + 1 < a.chunks ? each : (float)(a.pixels - at * a.chunk) * (float)a.per;
          all = join(all, {n, s[i].x, at < a.chunks ? s[i].y : 0.f});
        }
      }
    }
    for (int half = lanes / 2; half; half /= 2) {
      if (lane >= half && lane < 2 * half) part[threadIdx.x - half * here] = all;
      __syncthreads();
      if (lane < half) all = join(all, part[threadIdx.x]);
      __syncthreads();
    }
    if (lane == 0) {
      lds[g] = all.mean;
      lds[a.groups + g] = __builtin_amdgcn_rsqf(all.squares / all.n + a.eps);
    }
  }
  __syncthreads();
}

template <int DT, int EDGE, bool STREAM>
__global__ void group_norm_kernel(Args a) {
  typedef typename Type<DT>::T T;
  extern __shared__ float lds[];  // [2][groups] mean and 1 / deviation
  const int tx = threadIdx.x % a.vectors, ty = threadIdx.x / a.vectors, there = a.channels;
  const int c0 = EDGE == SHARED ? min(tx * V, a.channels - V) : tx * V;
  const T* const x = (const T*)a.x + blockIdx.y * a.x_b + c0;
  T* const out = (T*)a.out + blockIdx.y * a.out_b + c0;
  const uint32_t p0 = blockIdx.x * a.chunk, p1 = min(a.pixels, p0 + a.chunk), rows = a.rows;
  // What needs no statistics is asked for before them.  (Backwards: the thread's last pixels first.)
  constexpr int AT_ONCE = DT == HB_DTYPE_F32 ? 4 : 8;
  Raw<DT> raw[AT_ONCE];
  auto ask = [&](int i) {
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) raw[r] = load<DT, EDGE, STREAM>(x + (int64_t)(p0 + min(ty + (uint32_t)max(i - r, 0) * rows, p1 - p0 - 1)) * a.x_n, there);
  };
  int i = ((int)(p1 - p0) - ty + (int)rows - 1) / (int)rows - 1;
  ask(i);
  float mean[V], scale[V], shift[V];
#pragma unroll
  for (int k = 0; k < V; ++k) scale[k] = 1.f, shift[k] = 0.f;
  if (a.weight) unpack(load<DT, EDGE, false>((const T*)a.weight + c0, there), scale);
  if (a.bias) unpack(load<DT, EDGE, false>((const T*)a.bias + c0, there), shift);
  join_chunks(a, lds);
  int g = c0 / a.per, c = c0 - g * a.per;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    mean[k] = lds[g];
    scale[k] *= lds[a.groups + g];
    if (++c == a.per && g + 1 < a.groups) c = 0, ++g;
  }
  while (i >= 0) {
    float v[AT_ONCE][V];
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) unpack(raw[r], v[r]);
    const int done = i;
    i -= AT_ONCE;
    if (i >= 0) ask(i);
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {
      if (done < r) break;
#pragma unroll
      for (int k = 0; k < V; ++k) v[r][k] = activate((v[r][k] - mean[k]) * scale[k] + shift[k], a.silu);
      store<DT, EDGE, STREAM>(out + (int64_t)(p0 + ty + (done - r) * rows) * a.out_n, v[r], tx * V - c0, there);
    }
  }
}

// ------------------------------------------------------------------ groups that fit a workgroup
// W channels a load, up to UNITS loads a thread.  A few loads' and two barriers' time: 1 x 256 pixels x 512 channels, 32 groups
// 5.1 us from memory.
constexpr int UNITS = 2, FEW_THREADS = 1024;

template <int DT, int W>
__global__ __launch_bounds__(FEW_THREADS) void group_norm_few_kernel(Args a) {
  typedef typename Type<DT>::T T;
  __shared__ float parts[3][FEW_THREADS / 64];
  const int g = blockIdx.x, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const uint32_t across = a.per / W, all = a.pixels * across;  // loads of a pixel, and of the group
  const T* const x = (const T*)a.x + blockIdx.y * a.x_b + g * a.per;
  T* const out = (T*)a.out + blockIdx.y * a.out_b + g * a.per;
  typedef T Unit __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  auto widen = [](const Unit& u, float (&v)[W]) {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const T t = u[k];
      if constexpr (DT == HB_DTYPE_F32) v[k] = t;
      else v[k] = to_f<DT == HB_DTYPE_F16>(t);
    }
  };
  Unit raw[UNITS] = {}, weight[UNITS], bias[UNITS];
  uint32_t pixel[UNITS], channel[UNITS];
  bool there[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const uint32_t at = i * blockDim.x + threadIdx.x;
    there[i] = at < all;
    pixel[i] = at / across;
    channel[i] = (at - pixel[i] * across) * W;
    if (there[i]) raw[i] = *(const Unit*)(x + (int64_t)pixel[i] * a.x_n + channel[i]);
    if (a.weight) weight[i] = *(const Unit*)((const T*)a.weight + g * a.per + channel[i]);
    if (a.bias) bias[i] = *(const Unit*)((const T*)a.bias + g * a.per + channel[i]);
  }
  auto wave_total = [&](float s, float (&part)[FEW_THREADS / 64]) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    if ((threadIdx.x & 63) == 0) part[wave] = s;
  };
  auto total = [&](const float (&part)[FEW_THREADS / 64]) {
    float s = 0.f;
    for (int w = 0; w < waves; ++w) s += part[w];
    return s;
  };
  float v[UNITS][W], sum = 0.f, rest = 0.f, squares = 0.f;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    widen(raw[i], v[i]);
#pragma unroll
    for (int k = 0; k < W; ++k) sum += v[i][k];  // (zeros past the group's values)
  }
  wave_total(sum, parts[0]);
  __syncthreads();
  const float n = (float)all * W, mean = total(parts[0]) / n;
  // (the values' differences from the mean tell by how much its rounding missed theirs: a few values close together far
  // from zero would be off by the mean's last bit in their deviations)
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
#pragma unroll
    for (int k = 0; k < W; ++k) {
      v[i][k] = there[i] ? v[i][k] - mean : 0.f;
      rest += v[i][k];
      squares += v[i][k] * v[i][k];
    }
  wave_total(rest, parts[1]);
  wave_total(squares, parts[2]);
  __syncthreads();
  const float missed = total(parts[1]) / n, var = fmaxf(total(parts[2]) / n - missed * missed, 0.f);
  const float scale = __builtin_amdgcn_rsqf(var + a.eps);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    if (!there[i]) continue;
    float w[W], b[W];
    widen(weight[i], w);
    widen(bias[i], b);
    Unit u;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float y = activate((v[i][k] - missed) * (a.weight ? scale * w[k] : scale) + (a.bias ? b[k] : 0.f), a.silu);
      if constexpr (DT == HB_DTYPE_F32) u[k] = y;
      else u[k] = from_f<DT == HB_DTYPE_F16>(y);
    }
    *(Unit*)(out + (int64_t)pixel[i] * a.out_n + channel[i]) = u;
  }
}

// ------------------------------------------------------------------ launches
int64_t size_of(int dtype) { return dtype == HB_DTYPE_F32 ? 4 : 2; }

// Channels of a load of group_norm_few_kernel: the most that divide a group's.
int few_width(int per) { return per % 8 == 0 ? 8 : per % 4 == 0 ? 4 : per % 2 == 0 ? 2 : 1; }

// The kernels and chunks follow from an element's sizes alone, so that an image's result is the same in every batch: a
// batch of more workgroups than a launch takes (a grid holds fewer than 2^32 threads) goes in slices.
int32_t slice_of(int32_t batch, int64_t groups_of_one, int64_t threads) {
  return (int32_t)std::min<int64_t>(batch, ((1ll << 32) - 1) / (groups_of_one * threads));
}

// The elements from `first` on.
template <int DT>
Args from_element(Args a, int32_t first) {
  typedef typename Type<DT>::T T;
  a.x = (const T*)a.x + first * a.x_b;
  a.out = (T*)a.out + first * a.out_b;
  a.sums += (int64_t)first * a.chunks * a.groups;
  return a;
}

// Whether a workgroup holds a group.  One launch and two, 512 channels in 32 groups, us: 256 pixels 7.4, 10.6; 1024 8.7,
// 10.6; with groups twice and four times as large as a workgroup holds now 13.7, 10.9 and 30.4, 11.5.
bool few(int64_t pixels, int per) { return pixels * (per / few_width(per)) <= (int64_t)UNITS * FEW_THREADS; }

// Chunks of at least 16 KB, up to as many as there are CUs.
// us of 256, 512 chunks of 256 threads, and of 512 threads: 65536 pixels x 512 channels bf16 45.2, 47.3, 47.4, 47.0; 262144 x
// 256 fp32 142, 146, 150, 159, bf16 85, 88, 81, 87; 2048 x 2048 x 128 bf16 578, 550, 543, 534.  Of 16384 x 512 18.2, 20.4,
// 17.0, 23.8; 128 chunks 22.4: every workgroup of the second launch joins all chunks of its element.
//
// Twice as many of twice the threads where an element is large.  Once / twice, us, 128 channels: bf16 256 MB 131 / 135, 512
// 269 / 258, 640 367 / 344, 1024 576 / 533, 2048 1200 / 1137; fp32 576 MB 351 / 361, 640 398 / 393, 1024 684 / 633, 1536 1030 /
// 1028.  Rows that are neither whole lines nor some of one lose by it while they are short, 1024 MB: 20 channels bf16 912 /
// 928, 60 933 / 1040, 96 609 / 637, 330 709 / 739, fp32 60 868 / 947, 100 795 / 846; but 320 channels bf16 588 / 557, 500 697 / 672,
// 1002 751 / 720, fp32 250 734 / 726.  Fewer than eight channels are latency: 6 bf16 3400 / 1735.
bool large(int64_t bytes, int64_t row, int channels, int dtype) {
  return bytes > (dtype == HB_DTYPE_F32 ? LARGE_FLOAT_BYTES : LARGE_BYTES) &&
         (row % LINE == 0 || LINE % row == 0 || row >= 1000 || channels < V);
}

struct Chunks {
  int64_t pixels, count;
  int threads;
};
Chunks chunks_of(int64_t pixels, int channels, int dtype) {
  const int64_t row = channels * size_of(dtype);
  const int times = large(pixels * row, row, channels, dtype) ? 2 : 1;
  const int64_t count = std::clamp<int64_t>(pixels * row / CHUNK_BYTES, 1, 256 * times);
  const int64_t each = (pixels + count - 1) / count;
  return {each, (pixels + each - 1) / each, THREADS * times};
}

template <int DT, int W>
int launch_few(const Args& a, int32_t batch, hipStream_t st) {
  const int64_t units = (int64_t)a.pixels * (a.per / W);
  const int threads = (int)std::clamp<int64_t>((units + 63) / 64 * 64, 64, FEW_THREADS);
  const int32_t slice = slice_of(batch, a.groups, threads);
  for (int32_t b = 0; b < batch; b += slice) {
    hipLaunchKernelGGL((group_norm_few_kernel<DT, W>), dim3(a.groups, std::min(slice, batch - b)), dim3(threads), 0, st, from_element<DT>(a, b));
    HB_HIP(hipGetLastError());
  }
  return HB_OK;
}

template <int DT, int EDGE>
int launch_chunks(const Args& a, int32_t batch, bool stream_values, hipStream_t st) {
  const dim3 block(a.vectors * a.rows);
  const size_t lds = 2 * a.groups * sizeof(float);
  const int32_t slice = slice_of(batch, a.chunks, block.x);
  for (int32_t b = 0; b < batch; b += slice) {
    const dim3 grid(a.chunks, std::min(slice, batch - b));
    const Args part = from_element<DT>(a, b);
    hipLaunchKernelGGL((group_norm_sums_kernel<DT, EDGE>), grid, block, block.x * V * 2 * sizeof(float), st, part);
    HB_HIP(hipGetLastError());
    if (stream_values) hipLaunchKernelGGL((group_norm_kernel<DT, EDGE, true>), grid, block, lds, st, part);
    else hipLaunchKernelGGL((group_norm_kernel<DT, EDGE, false>), grid, block, lds, st, part);
    HB_HIP(hipGetLastError());
  }
  return HB_OK;
}

template <int DT>
int launch(Args& a, int32_t batch, hipStream_t st) {
  if (few(a.pixels, a.per)) {
    switch (few_width(a.per)) {
      case 8: return launch_few<DT, 8>(a, batch, st);
      case 4: return launch_few<DT, 4>(a, batch, st);
      case 2: return launch_few<DT, 2>(a, batch, st);
      default: return launch_few<DT, 1>(a, batch, st);
    }
  }
  // (an expanded x as well, whose image the caches would hold: through them 64 x 16384 x 256 264 -> 259 us, 256 x 4096 x 256 394 ->
  // 382, but 4 x 262144 x 256 235 -> 240)
  const bool stream_values = 2 * (int64_t)batch * a.pixels * a.channels * size_of(DT) > CACHE_BYTES;
  if (a.channels < V) return launch_chunks<DT, SHORT>(a, batch, stream_values, st);
  return a.channels % V ? launch_chunks<DT, SHARED>(a, batch, stream_values, st) : launch_chunks<DT, EVEN>(a, batch, stream_values, st);
}

}  // namespace
}  // namespace hb

using namespace hb;

namespace {
int check_sizes(int32_t batch, int64_t pixels, int32_t channels, int32_t groups, int32_t dtype) {
  HB_REQUIRE(batch > 0 && batch <= 65535 && pixels > 0 && pixels < (1ll << 31), "batch must be in [1, 65535] and pixels in [1, 2^31)");
  HB_REQUIRE(channels > 0 && channels <= MAX_CHANNELS, "channels must be in [1, %d] (got %d)", MAX_CHANNELS, channels);
  HB_REQUIRE(groups > 0 && channels % groups == 0, "groups must divide the channels");
  HB_REQUIRE(dtype == HB_DTYPE_BF16 || dtype == HB_DTYPE_F16 || dtype == HB_DTYPE_F32, "dtype must be bf16, fp16 or fp32");
  return HB_OK;
}
}  // namespace

extern "C" int64_t hb_group_norm_workspace_bytes(int32_t batch, int64_t pixels, int32_t channels, int32_t groups, int32_t dtype) {
  if (check_sizes(batch, pixels, channels, groups, dtype) != HB_OK) return -1;
  if (few(pixels, channels / groups)) return 0;
  return batch * chunks_of(pixels, channels, dtype).count * groups * (int64_t)sizeof(float2);
}

extern "C" int hb_group_norm(int32_t batch, int64_t pixels, int32_t channels, int32_t groups, int32_t dtype, int32_t silu,
                             float eps, const void* x, int64_t x_batch_stride, int64_t x_pixel_stride, const void* weight,
                             const void* bias, void* out, int64_t out_batch_stride, int64_t out_pixel_stride,
                             void* workspace, int64_t workspace_bytes, hb_stream_t stream) {
  HB_REQUIRE(x && out, "null pointer argument");
  const int rc = check_sizes(batch, pixels, channels, groups, dtype);
  if (rc) return rc;
  HB_REQUIRE(silu == 0 || silu == 1, "silu must be 0 or 1");
  // (the root takes a smaller number for zero: a group without deviation would be NaN)
  HB_REQUIRE(eps >= 0x1p-126f, "eps must be at least 2^-126");
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
  const int64_t need = hb_group_norm_workspace_bytes(batch, pixels, channels, groups, dtype);
  if (need) {
    HB_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need, "the workspace must hold %lld bytes, 8-byte aligned", (long long)need);
    const Chunks c = chunks_of(pixels, channels, dtype);
    a.sums = (float2*)workspace;
    a.chunk = (uint32_t)c.pixels;
    a.chunks = (uint32_t)c.count;
    a.rows = std::max(1, c.threads / a.vectors);
  }
  switch (dtype) {
    case HB_DTYPE_BF16: return launch<HB_DTYPE_BF16>(a, batch, stream);
    case HB_DTYPE_F16: return launch<HB_DTYPE_F16>(a, batch, stream);
    default: return launch<HB_DTYPE_F32>(a, batch, stream);
  }
}
