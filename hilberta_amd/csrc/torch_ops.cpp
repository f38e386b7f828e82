// The torch operators of namespace hilberta_hip, over the C ABI (include/hilberta_hip.h).
//
// The reference launches its kernels as framework-visible Triton launches (hilberta/paired_kernel.py
// :181-204, hilberta/sparse_kernel.py:315-339) and gathers with index_select (hilberta/flux_adapter.py
// :209-212, :243).  Registered here natively, an operator call costs the host a few microseconds; as
// Python functions behind torch's dispatcher the attention operator took 22 us and a gather 16.5 us,
// more than the kernels of a 512 px attention call or a latents gather.  The shape-only (fake)
// implementations and the CPU kernel of pair_rows, which is plan setup, are in hilberta_amd/ops.py.
#include <ATen/ATen.h>
#include <ATen/DeviceGuard.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <initializer_list>
#include <limits>
#include <map>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/hilberta_hip.h"

namespace {

using at::Tensor;

// Key blocks per row hb_pair_rows pairs.
constexpr int64_t PAIR_MAX_BLOCKS = 16384;
constexpr int64_t MIN_WORKSPACE = 1 << 16;
// Features of 8-bit rows: a sum of so many products fits 32 bits.
constexpr int64_t MAX_FEATURES = 1 << 17;

void check(int rc, const char* name) {
  if (rc == 0) return;
  if (rc == 1) TORCH_CHECK_VALUE(false, name, ": ", hb_last_error());
  TORCH_CHECK(false, name, ": ", hb_last_error());
}

int32_t i32(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= std::numeric_limits<int32_t>::min() && v <= std::numeric_limits<int32_t>::max(),
                    name, " does not fit 32 bits");
  return static_cast<int32_t>(v);
}

hipStream_t stream_of(const at::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

// ------------------------------------------------------------------ attention workspaces
// One workspace per (device, stream): the persistent kernel's work-queue counters (zero-filled once;
// every launch leaves them at zero) and the partial results of split global query tiles.  Launches
// that may overlap in time are on different streams and so never share one.  A call launches two
// kernels over its workspace, so threads of one stream take turns: each holds the workspace (Lease)
// until both are enqueued, or the second thread's first kernel could come between them.  A captured
// launch gets a workspace of its own from the capture's private pool, zero-filled on every replay.
class Workspaces {
  struct Held {
    std::mutex launching;
    Tensor tensor;
  };

 public:
  struct Lease {
    Tensor tensor;
    std::shared_ptr<Held> held;
    std::unique_lock<std::mutex> turn;
  };

  Lease get(const at::Device& device, int64_t need) {
    const auto options = at::TensorOptions().dtype(at::kByte).device(device);
    const int64_t bytes = std::max(need, MIN_WORKSPACE);
    const hipStream_t stream = stream_of(device);
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing(stream, &status) == hipSuccess, "stream capture query failed");
    if (status != hipStreamCaptureStatusNone) return {at::zeros({bytes}, options), nullptr, {}};
    Lease lease;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      std::shared_ptr<Held>& held = cache_[{device.index(), reinterpret_cast<int64_t>(stream)}];
      if (!held) held = std::make_shared<Held>();
      lease.held = held;
    }
    lease.turn = std::unique_lock<std::mutex>(lease.held->launching);
    Tensor& tensor = lease.held->tensor;
    if (!tensor.defined() || tensor.numel() < need) tensor = at::zeros({bytes}, options);
    lease.tensor = tensor;
    return lease;
  }

  std::vector<int64_t> keys() {
    const std::lock_guard<std::mutex> lock(mutex_);
    std::vector<int64_t> out;
    for (const auto& [key, held] : cache_) {
      out.push_back(key.first);
      out.push_back(key.second);
    }
    return out;
  }

  void clear() {
    std::map<Key, std::shared_ptr<Held>> gone;
    const std::lock_guard<std::mutex> lock(mutex_);
    gone.swap(cache_);
  }

 private:
  using Key = std::pair<int64_t, int64_t>;
  std::mutex mutex_;
  std::map<Key, std::shared_ptr<Held>> cache_;
};

// Never destroyed: at process exit the allocator behind the tensors may be gone first.
Workspaces& workspaces() {
  static Workspaces* w = new Workspaces;
  return *w;
}

Tensor attention_workspace(at::Device device, int64_t need) {
  TORCH_CHECK_VALUE(device.is_cuda(), "workspaces live on a HIP device");
  if (!device.has_index()) device = at::Device(at::kCUDA, c10::hip::current_device());
  const at::OptionalDeviceGuard guard(device);
  return workspaces().get(device, need).tensor;
}

std::vector<int64_t> workspace_keys() { return workspaces().keys(); }
void clear_workspaces() { workspaces().clear(); }

// The C ABI this library was compiled against (ops.py compares it before it binds the operators).
int64_t abi_version() { return HB_ABI_VERSION; }

// ------------------------------------------------------------------ operators
struct Shape {
  int32_t batch, heads, tokens, dim, dtype;
  int64_t strides[12];
};

Shape shape_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.sizes() == q.sizes() && v.sizes() == q.sizes() && out.sizes() == q.sizes(),
                    "Q/K/V/out must have equal [B,H,N,D] shapes");
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
                    "Q/K/V must be bf16 or fp16");
  Shape s{i32(q.size(0), "batch"), i32(q.size(1), "heads"), i32(q.size(2), "tokens"),
          i32(q.size(3), "head_dim"), q.scalar_type() == at::kHalf ? HB_DTYPE_F16 : HB_DTYPE_BF16, {}};
  int i = 0;
  for (const Tensor* t : {&q, &k, &v, &out})
    for (int d = 0; d < 3; ++d) s.strides[i++] = t->stride(d);
  return s;
}

float* lse_ptr(const std::optional<Tensor>& lse) {
  return lse.has_value() && lse->defined() ? static_cast<float*>(lse->data_ptr()) : nullptr;
}

Workspaces::Lease workspace_for(const Tensor& q, const Shape& s, int32_t global_tokens, int32_t width,
                     int32_t key_block, int32_t paired, bool all_queries) {
  const int64_t need = hb_attention_workspace_bytes(s.batch, s.heads, s.tokens, s.dim, global_tokens, width,
                                                    key_block, paired, all_queries);
  check(need < 0 ? 1 : 0, "hb_attention_workspace_bytes");
  return workspaces().get(q.device(), need);
}

void paired_launch(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
                   const std::optional<Tensor>& lse, const Tensor& ids, const Tensor& flags,
                   const Tensor& counts, int64_t global_tokens, int64_t key_block, double scale_log2,
                   bool all_queries, int64_t num_groups) {
  const Shape s = shape_of(q, k, v, out);
  const int32_t width = i32(ids.size(1), "table width"), G = i32(global_tokens, "global_tokens"),
                kb = i32(key_block, "key_block_size");
  const auto ws = workspace_for(q, s, G, width, kb, 1, all_queries);
  check(hb_paired_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_ptr(lse), s.strides, s.batch,
                      s.heads, s.tokens, s.dim, s.dtype, static_cast<const int32_t*>(ids.data_ptr()),
                      static_cast<const int32_t*>(flags.data_ptr()),
                      static_cast<const int32_t*>(counts.data_ptr()), width, G, kb, all_queries,
                      static_cast<float>(scale_log2), ws.tensor.data_ptr(), ws.tensor.numel(),
                      i32(num_groups, "num_groups"), stream_of(q.device())),
        "hb_paired_fwd");
}

// hb_paired_fwd on the current stream (replaces the _paired_fwd launch, paired_kernel.py:181-204).
void paired_fwd(const Tensor& q, const Tensor& k, const Tensor& v, Tensor out, std::optional<Tensor> lse,
                const Tensor& ids, const Tensor& flags, const Tensor& counts, int64_t global_tokens,
                int64_t key_block, double scale_log2, bool all_queries, int64_t num_groups) {
  const at::OptionalDeviceGuard guard(q.device());
  paired_launch(q, k, v, out, lse, ids, flags, counts, global_tokens, key_block, scale_log2, all_queries,
                num_groups);
}

// hb_pair_rows: rows 2r and 2r + 1 of an unpaired table become paired row r, ascending and
// zero-padded (paired_metadata.py:26-51); an odd row count is paired from the end.
std::tuple<Tensor, Tensor, Tensor> pair_rows(const Tensor& ids, const Tensor& counts, int64_t total_blocks,
                                             int64_t key_block, int64_t paired_width) {
  TORCH_CHECK_VALUE(ids.scalar_type() == at::kInt && counts.scalar_type() == at::kInt && ids.dim() == 2 &&
                        counts.dim() == 1 && counts.size(0) == ids.size(0) && ids.is_contiguous() &&
                        counts.is_contiguous() && ids.device() == counts.device(),
                    "tables must be contiguous int32 kv_indices [rows, width] and kv_counts [rows] on one device");
  const at::OptionalDeviceGuard guard(ids.device());
  const int64_t rows = ids.size(0), prows = (rows + 1) / 2;
  Tensor out = at::empty({prows, paired_width}, ids.options()), flags = at::empty_like(out);
  Tensor out_counts = at::empty({prows}, ids.options());
  check(hb_pair_rows(static_cast<const int32_t*>(ids.data_ptr()), static_cast<const int32_t*>(counts.data_ptr()),
                     i32(rows, "rows"), i32(ids.size(1), "width"), i32(total_blocks, "total_blocks"),
                     i32(key_block, "key_block_size"), static_cast<int32_t*>(out.data_ptr()),
                     static_cast<int32_t*>(flags.data_ptr()), static_cast<int32_t*>(out_counts.data_ptr()),
                     i32(paired_width, "paired_width"), nullptr, stream_of(ids.device())),
        "hb_pair_rows");
  return {out, flags, out_counts};
}

// Unpaired 64-query tables (replaces the _block_sparse_fwd launch, sparse_kernel.py:315-339).
//
// With at most PAIR_MAX_BLOCKS key blocks, rows 2r, 2r + 1 are merged on the device, as pair_metadata
// does (paired_metadata.py:26-51), and run on hb_paired_fwd: a 128-query item keeps two waves per
// SIMD busy where a 64-query item keeps one (1.7-1.85x faster).  An odd row count is paired from the
// end, its first paired row carrying an empty half that reaches into the global prefix and is never
// stored; a global prefix that is an odd multiple of 64 leaves a last global tile whose upper half is
// never stored either.  Every query sees the same key blocks in the same ascending order with the
// same arithmetic; the other half's blocks are masked to exact zeros.  The paired tables are padded
// to min(2 * width, N / 64) entries, which needs no host synchronisation.  Longer sequences run as
// they are on hb_block_sparse_fwd.
void sparse_fwd(const Tensor& q, const Tensor& k, const Tensor& v, Tensor out, std::optional<Tensor> lse,
                const Tensor& ids, const Tensor& counts, int64_t global_tokens, double scale_log2,
                bool all_queries, int64_t num_groups) {
  const at::OptionalDeviceGuard guard(q.device());
  const Shape s = shape_of(q, k, v, out);
  const int64_t blocks = s.tokens / 64;
  if (blocks <= PAIR_MAX_BLOCKS) {
    const auto [pids, pflags, pcounts] = pair_rows(ids, counts, blocks, 64, std::min(2 * ids.size(1), blocks));
    paired_launch(q, k, v, out, lse, pids, pflags, pcounts, global_tokens, 64, scale_log2, all_queries, num_groups);
    return;
  }
  const int32_t width = i32(ids.size(1), "table width"), G = i32(global_tokens, "global_tokens");
  const auto ws = workspace_for(q, s, G, width, 64, 0, all_queries);
  check(hb_block_sparse_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_ptr(lse), s.strides,
                            s.batch, s.heads, s.tokens, s.dim, s.dtype, static_cast<const int32_t*>(ids.data_ptr()),
                            static_cast<const int32_t*>(counts.data_ptr()), width, G, 64, all_queries,
                            static_cast<float>(scale_log2), ws.tensor.data_ptr(), ws.tensor.numel(),
                            i32(num_groups, "num_groups"), stream_of(q.device())),
        "hb_block_sparse_fwd");
}

// One stride walking every index of the dims before `dim`: {count, stride}, stride -1 if none does.
std::pair<int64_t, int64_t> outer_walk(const Tensor& x, int64_t dim) {
  int64_t outer = 1, last = 0, step = -1;  // step: what the next dim outwards must advance by
  for (int64_t d = 0; d < dim; ++d) outer *= x.size(d);
  if (outer <= 1) return {outer, 0};
  for (int64_t d = dim - 1; d >= 0; --d) {
    if (x.size(d) <= 1) continue;
    if (step < 0) last = x.stride(d);
    else if (x.stride(d) != step) return {outer, -1};
    step = x.stride(d) * x.size(d);
  }
  return {outer, last};
}

// x.index_select(dim, index) by hb_gather_rows (flux_adapter.py:209-212, :243), bit for bit; the
// dims after `dim` must be contiguous.
Tensor gather_rows(const Tensor& input, int64_t dim, const Tensor& index) {
  const int64_t nd = input.dim();
  TORCH_CHECK_INDEX(nd > 0 && dim >= -nd && dim < nd, "dim out of range");
  if (dim < 0) dim += nd;
  TORCH_CHECK_VALUE(index.dim() == 1 && index.scalar_type() == at::kLong && index.device() == input.device(),
                    "index must be a 1-D int64 tensor on x's device");
  int64_t row = 1;
  for (int64_t d = nd - 1; d > dim; --d) {
    TORCH_CHECK_VALUE(input.size(d) <= 1 || input.stride(d) == row,
                      "index_select_rows needs the dims after `dim` to be contiguous");
    row *= input.size(d);
  }
  const at::OptionalDeviceGuard guard(input.device());
  Tensor x = input;
  auto [outer, src_outer] = outer_walk(x, dim);
  if (src_outer < 0) {
    x = x.contiguous();
    std::tie(outer, src_outer) = outer_walk(x, dim);
  }
  const Tensor idx = index.contiguous();
  auto sizes = x.sizes().vec();
  sizes[dim] = idx.numel();
  Tensor out = at::empty(sizes, x.options());
  const int64_t es = x.element_size();
  check(hb_gather_rows(x.data_ptr(), out.data_ptr(), static_cast<const int64_t*>(idx.data_ptr()), idx.numel(),
                       outer, src_outer * es, idx.numel() * row * es, x.stride(dim) * es, row * es, row * es,
                       x.size(dim), nullptr, stream_of(x.device())),
        "hb_gather_rows");
  return out;
}

// ------------------------------------------------------------------ 8-bit linear layers
// The operators' arguments are checked here, on any device, and then refused unless they are on a HIP one.
int32_t type_of(at::ScalarType t, const char* name) {
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf, name, " must be bf16 or fp16");
  return t == at::kHalf ? HB_DTYPE_F16 : HB_DTYPE_BF16;
}

void require_hip(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "HIP entry points take device tensors on one CUDA (HIP) device");
}

void one_device(const Tensor& first, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == first.device(), "all tensors must be on one device");
}

const Tensor& value_or_none(const std::optional<Tensor>& t) {
  static const Tensor* none = new Tensor;
  return t.has_value() ? *t : *none;
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Leading dimensions of t, all but the last, as {batch, rows, batch stride, row stride}.
struct Rows {
  int64_t batch, rows, batch_stride, row_stride;
};

Rows rows_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 2 || t.dim() == 3, name, " must be [rows, columns] or [batch, rows, columns]");
  TORCH_CHECK_VALUE(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have a contiguous last dimension");
  if (t.dim() == 2) return {1, t.size(0), 0, t.stride(0)};
  return {t.size(0), t.size(1), t.stride(0), t.stride(1)};
}

// [begin, end) of a view's bytes.
std::pair<const char*, const char*> bytes_of(const Tensor& t) {
  int64_t extent = 1;
  for (int64_t d = 0; d < t.dim(); ++d) extent += (t.size(d) - 1) * t.stride(d);
  const char* begin = static_cast<const char*>(t.data_ptr());
  return {begin, begin + (t.numel() ? extent * t.element_size() : 0)};
}

// What is written has places of its own: no two of its values share one, and no input lies among them.
void check_written(const Tensor& out, const char* name, std::initializer_list<const Tensor*> inputs) {
  if (!out.numel()) return;
  c10::SmallVector<std::pair<int64_t, int64_t>, 5> dims;
  for (int64_t d = 0; d < out.dim(); ++d)
    if (out.size(d) > 1) dims.emplace_back(out.stride(d), out.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t extent = 1;
  for (const auto& [stride, size] : dims) {
    TORCH_CHECK_VALUE(stride >= extent, name, " must have positive, non-overlapping strides");
    extent += (size - 1) * stride;
  }
  const auto [begin, end] = bytes_of(out);
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->numel()) continue;
    const auto [first, last] = bytes_of(*t);
    TORCH_CHECK_VALUE(!(begin < last && first < end), name, " cannot alias the inputs");
  }
}

// Whether two views of rows may share a value: no where their bytes lie apart, or where row ranges or column
// blocks of one buffer do.
bool may_overlap(const Tensor& a, const Tensor& b) {
  if (!a.numel() || !b.numel()) return false;
  const auto [a0, a1] = bytes_of(a);
  const auto [b0, b1] = bytes_of(b);
  if (a1 <= b0 || b1 <= a0) return false;
  const Rows ra = rows_of(a, "rows"), rb = rows_of(b, "rows");
  const int64_t size = a.element_size(), delta = b0 - a0;
  if (b.element_size() != size || delta % size) return true;
  // Within a period of both views, one takes its first `na` elements and the other `nb` from d on.
  const auto apart = [&](int64_t period, int64_t na, int64_t nb) {
    const int64_t d = ((delta / size) % period + period) % period;
    return d >= na && d + nb <= period;
  };
  const bool many = a.dim() == 3 && b.dim() == 3 && (ra.batch > 1 || rb.batch > 1);
  const int64_t row = ra.row_stride, all = many ? ra.batch_stride : 0;
  if (rb.row_stride != row || row <= 0 || (many && (rb.batch_stride != all || all <= 0))) return true;
  if ((!many || all % row == 0) && apart(row, a.size(-1), b.size(-1))) return false;
  return !(many && apart(all, (ra.rows - 1) * row + a.size(-1), (rb.rows - 1) * row + b.size(-1)));
}

// Whether two views of one shape are the same places in the same order.
bool same_places(const Tensor& a, const Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

// Checks of 8-bit rows [.., padded] with their scales; returns padded.
int64_t check_int8(const Tensor& q, const Tensor& scale, const char* name) {
  TORCH_CHECK_VALUE(q.dim() >= 2 && q.scalar_type() == at::kChar && q.is_contiguous() && q.size(-1) > 0 &&
                        q.size(-1) % 64 == 0,
                    name, " must be contiguous int8 rows of a multiple of 64 columns");
  TORCH_CHECK_VALUE(scale.scalar_type() == at::kFloat && scale.is_contiguous() &&
                        scale.sizes() == q.sizes().slice(0, q.dim() - 1),
                    name, " must have one contiguous float32 scale a row");
  return q.size(-1);
}

// Columns of 8-bit rows of `features` values.
int64_t padded_features(int64_t features) { return (features + 63) / 64 * 64; }

// An unwritten tensor on x's device.  (Not through the dispatcher: it takes as long as the allocation does, and
// the short calls here are the host's.)
Tensor new_tensor(const Tensor& x, at::IntArrayRef sizes, at::ScalarType dtype) {
  if (!x.is_cuda()) return at::empty(sizes, x.options().dtype(dtype));
  return Tensor(at::detail::empty_cuda(sizes, dtype, x.device(), std::nullopt));
}

// Unwritten 8-bit rows for x [.., features], and their scales.
std::tuple<Tensor, Tensor> new_int8_rows(const Tensor& x) {
  c10::SmallVector<int64_t, 3> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = padded_features(sizes.back());
  Tensor q = new_tensor(x, sizes, at::kChar);
  sizes.pop_back();
  return {std::move(q), new_tensor(x, sizes, at::kFloat)};
}

// hb_int8_rows: 16-bit rows to 8-bit rows and their scales.
std::tuple<Tensor, Tensor> int8_rows(const Tensor& x) {
  const int32_t dtype = type_of(x.scalar_type(), "rows");
  TORCH_CHECK_VALUE((x.dim() == 2 || x.dim() == 3) && x.size(-1) > 0 && x.size(-1) <= MAX_FEATURES,
                    "rows must be [rows, features] or [B, rows, features] of 1 to ", MAX_FEATURES, " features");
  const Rows r = rows_of(x, "rows");
  require_hip(x);
  const at::OptionalDeviceGuard guard(x.device());
  auto [q, scale] = new_int8_rows(x);
  if (scale.numel())
    check(hb_int8_rows(x.data_ptr(), r.batch_stride, r.row_stride, i32(r.batch, "batch"), i32(r.rows, "rows"),
                       i32(x.size(-1), "features"), i32(q.size(-1), "padded"), dtype, static_cast<int8_t*>(q.data_ptr()),
                       static_cast<float*>(scale.data_ptr()), stream_of(x.device())),
          "hb_int8_rows");
  return {std::move(q), std::move(scale)};
}

struct AdaSet {
  const Tensor &x, &shift, &scale;
  const std::optional<Tensor>&y, &gate, &x_out;
};

// hb_int8_adaln of one or two row sets; their 8-bit rows and scales.
std::array<Tensor, 4> int8_adaln_sets(std::initializer_list<AdaSet> sets, double eps) {
  void* pointers[16];
  int64_t strides[16];
  int32_t rows[2];
  const AdaSet& s0 = *sets.begin();
  std::array<Tensor, 4> made;
  const int32_t dtype = type_of(s0.x.scalar_type(), "rows");
  const int64_t batch = s0.x.dim() == 3 ? s0.x.size(0) : 1, hidden = s0.x.dim() ? s0.x.size(-1) : 0;
  TORCH_CHECK_VALUE(hidden > 0 && hidden % 8 == 0 && hidden <= 8192, "hidden must be a multiple of 8 up to 8192");
  const int64_t padded = padded_features(hidden);
  int i = 0;
  for (const AdaSet& s : sets) {
    const Tensor &y = value_or_none(s.y), &gate = value_or_none(s.gate), &x_out = value_or_none(s.x_out);
    TORCH_CHECK_VALUE(s.x.dim() == 3 && s.x.size(0) == batch && s.x.size(2) == hidden &&
                          s.x.scalar_type() == s0.x.scalar_type(),
                      "x must be [B, rows, hidden], both row sets of one batch, hidden size and dtype");
    TORCH_CHECK_VALUE(y.defined() == gate.defined(), "y and gate are given together");
    TORCH_CHECK_VALUE(!x_out.defined() || y.defined(), "x_out is written only with a residual update");
    for (const Tensor* t : {&y, &x_out})
      TORCH_CHECK_VALUE(!t->defined() || (t->sizes() == s.x.sizes() && t->scalar_type() == s.x.scalar_type()),
                        "y and x_out must be like x");
    for (const Tensor* t : {&s.shift, &s.scale, &gate})
      TORCH_CHECK_VALUE(!t->defined() || (t->dim() == 2 && t->size(0) == batch && t->size(1) == hidden &&
                                          (hidden <= 1 || t->stride(1) == 1) && t->scalar_type() == s.x.scalar_type()),
                        "shift/scale/gate must be [B, hidden] views with a contiguous last dim");
    TORCH_CHECK_VALUE(batch == 1 || s.shift.stride(0) == s.scale.stride(0), "shift and scale must share one batch stride");
    const Rows rx = rows_of(s.x, "x"), ry = y.defined() ? rows_of(y, "y") : Rows{},
               ro = x_out.defined() ? rows_of(x_out, "x_out") : Rows{};
    if (x_out.defined()) {
      for (const AdaSet& other : sets) {
        check_written(x_out, "x_out", {&other.shift, &other.scale, &value_or_none(other.gate)});
        // (a row is read before it is written, by one wave: x_out may be this set's x or y)
        const bool own = &other == &s;
        for (const Tensor* t : {&other.x, &value_or_none(other.y)})
          TORCH_CHECK_VALUE(!t->defined() || (own && same_places(x_out, *t)) || !may_overlap(x_out, *t),
                            "x_out must be x itself or lie apart from the rows read");
        TORCH_CHECK_VALUE(own || !other.x_out.has_value() || !may_overlap(x_out, *other.x_out),
                          "both sets' x_out must lie apart");
      }
    }
    one_device(s0.x, {&s.x, &s.shift, &s.scale, &y, &gate, &x_out});
    if (!s.x.numel()) continue;  // (a set without rows takes no part in the launch)
    void* p[8] = {pointer(s.x), pointer(y), pointer(gate), pointer(x_out), pointer(s.shift), pointer(s.scale), nullptr, nullptr};
    // (a stride of a dimension of one says nothing)
    const int64_t one = batch == 1 ? 0 : 1;
    const int64_t st[8] = {one * rx.batch_stride, rx.rows == 1 ? 0 : rx.row_stride, one * ry.batch_stride,
                           rx.rows == 1 ? 0 : ry.row_stride, gate.defined() ? one * gate.stride(0) : 0,
                           one * ro.batch_stride, rx.rows == 1 ? 0 : ro.row_stride, one * s.shift.stride(0)};
    std::copy(p, p + 8, pointers + 8 * i);
    std::copy(st, st + 8, strides + 8 * i);
    rows[i++] = i32(rx.rows, "rows");
  }
  require_hip(s0.x);
  const at::OptionalDeviceGuard guard(s0.x.device());
  int count = 0;
  i = 0;
  for (const AdaSet& s : sets) {
    std::tie(made[2 * i], made[2 * i + 1]) = new_int8_rows(s.x);
    if (s.x.numel()) {
      pointers[8 * count + 6] = made[2 * i].data_ptr();
      pointers[8 * count++ + 7] = made[2 * i + 1].data_ptr();
    }
    ++i;
  }
  if (!count) return made;
  check(hb_int8_adaln(count, i32(batch, "batch"), rows, i32(hidden, "hidden"), i32(padded, "padded"), dtype,
                      static_cast<float>(eps), pointers, strides, stream_of(s0.x.device())),
        "hb_int8_adaln");
  return made;
}

using Maybe = std::optional<Tensor>;

std::tuple<Tensor, Tensor> int8_adaln(const Tensor& x, const Tensor& shift, const Tensor& scale, const Maybe& y,
                                      const Maybe& gate, Maybe x_out, double eps) {
  auto made = int8_adaln_sets({{x, shift, scale, y, gate, x_out}}, eps);
  return {std::move(made[0]), std::move(made[1])};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> int8_adaln_pair(
    const Tensor& x, const Tensor& shift, const Tensor& scale, const Maybe& y, const Maybe& gate, Maybe x_out,
    const Tensor& x2, const Tensor& shift2, const Tensor& scale2, const Maybe& y2, const Maybe& gate2, Maybe x_out2,
    double eps) {
  auto made = int8_adaln_sets({{x, shift, scale, y, gate, x_out}, {x2, shift2, scale2, y2, gate2, x_out2}}, eps);
  return {std::move(made[0]), std::move(made[1]), std::move(made[2]), std::move(made[3])};
}

// Checks of a weight [columns, padded] with its scales and bias.
void check_weight(const Tensor& w, const Tensor& scale, const Tensor& bias, int64_t padded, int64_t columns,
                  at::ScalarType dtype) {
  TORCH_CHECK_VALUE(w.dim() == 2 && check_int8(w, scale, "weight") == padded && w.size(0) == columns,
                    "weight must be [columns, padded features], as the rows are padded");
  TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == columns && bias.is_contiguous() &&
                                        bias.scalar_type() == dtype),
                    "bias must be a contiguous [columns] tensor of the output's dtype");
}

struct LinearSet {
  const Tensor &q, &scale, &weight, &weight_scale;
  const std::optional<Tensor>& bias;
  const Tensor& out;
};

void int8_linear_sets(std::initializer_list<LinearSet> sets, bool gelu) {
  void* pointers[12];
  int64_t strides[4];
  int32_t rows[2];
  const LinearSet& s0 = *sets.begin();
  const int32_t dtype = type_of(s0.out.scalar_type(), "out");
  const int64_t padded = check_int8(s0.q, s0.scale, "rows");
  const int64_t batch = s0.out.dim() == 3 ? s0.out.size(0) : 1;
  int i = 0;
  for (const LinearSet& s : sets) {
    const Tensor& bias = value_or_none(s.bias);
    const Rows r = rows_of(s.out, "out");
    TORCH_CHECK_VALUE(check_int8(s.q, s.scale, "rows") == padded && r.batch == batch &&
                          s.out.scalar_type() == s0.out.scalar_type() && s.out.size(-1) == s0.out.size(-1),
                      "both row sets must share batch, features, columns and dtype");
    TORCH_CHECK_VALUE(s.q.sizes().slice(0, s.q.dim() - 1) == s.out.sizes().slice(0, s.out.dim() - 1),
                      "out must have the rows' leading dimensions");
    check_weight(s.weight, s.weight_scale, bias, padded, s.out.size(-1), s.out.scalar_type());
    for (const LinearSet& o : sets) {
      check_written(s.out, "out", {&o.q, &o.scale, &o.weight, &o.weight_scale, &value_or_none(o.bias)});
      TORCH_CHECK_VALUE(&o == &s || !may_overlap(s.out, o.out), "both outputs must lie apart");
    }
    one_device(s0.q, {&s.q, &s.scale, &s.weight, &s.weight_scale, &bias, &s.out});
    if (!s.out.numel()) continue;  // (a set without rows takes no part in the launch)
    void* p[6] = {pointer(s.q), pointer(s.scale), pointer(s.weight), pointer(s.weight_scale), pointer(bias), pointer(s.out)};
    std::copy(p, p + 6, pointers + 6 * i);
    strides[2 * i] = batch == 1 ? 0 : r.batch_stride;
    strides[2 * i + 1] = r.rows == 1 ? 0 : r.row_stride;
    rows[i++] = i32(r.rows, "rows");
  }
  require_hip(s0.q);
  if (!i) return;
  const at::OptionalDeviceGuard guard(s0.q.device());
  check(hb_int8_linear(i, i32(batch, "batch"), rows, i32(s0.out.size(-1), "columns"), i32(padded, "padded"), dtype, gelu,
                       pointers, strides, stream_of(s0.q.device())),
        "hb_int8_linear");
}

void int8_linear_out(const Tensor& q, const Tensor& scale, const Tensor& weight, const Tensor& weight_scale,
                     const Maybe& bias, Tensor out, bool gelu) {
  int8_linear_sets({{q, scale, weight, weight_scale, bias, out}}, gelu);
}

Tensor int8_linear(const Tensor& q, const Tensor& scale, const Tensor& weight, const Tensor& weight_scale,
                   const Maybe& bias, at::ScalarType dtype, bool gelu) {
  type_of(dtype, "rows");
  TORCH_CHECK_VALUE((q.dim() == 2 || q.dim() == 3) && weight.dim() == 2,
                    "rows must be [rows, padded] or [B, rows, padded] and weight [columns, padded]");
  c10::SmallVector<int64_t, 3> sizes(q.sizes().begin(), q.sizes().end());
  sizes.back() = weight.size(0);
  Tensor out = new_tensor(q, sizes, dtype);
  int8_linear_out(q, scale, weight, weight_scale, bias, out, gelu);
  return out;
}

// Whether a few 16-bit rows take one launch (hb_int8_linear_rows): where its workgroups, which quantize the rows each
// for itself, run all at once, and ask for the weight as fast as the product of 8-bit rows does: a weight up to 48 MB,
// or enough workgroups.  Rows x features x columns, us for two launches and one: 1 x 512 x 2048 12.4, 6.0; 1 x 3072 x
// 18432 16.1, 11.5; 5 x 3072 x 18432 16.5, 12.8; 32 x 512 x 18432 12.3, 11.2; 1 x 12288 x 3072 21.7, 14.9; on the other
// side 1 x 8192 x 8192 17.4, 20.7; 30 x 512 x 30000 12.3, 16.4.
bool one_launch(int64_t rows, int64_t features, int64_t columns) {
  return rows <= 32 && features >= 8 && rows * ((features + 127) / 128 * 128) <= HB_INT8_FEW_VALUES && columns <= 24576 &&
         (padded_features(features) * columns <= (48 << 20) || columns >= 14336);
}

// int8_rows and int8_linear in one call: a short layer's time is the host's.
Tensor int8_linear_rows(const Tensor& x, const Tensor& weight, const Tensor& weight_scale, const Maybe& bias, bool gelu) {
  const int64_t count = x.dim() ? x.numel() / std::max<int64_t>(x.size(-1), 1) : 0, features = x.dim() ? x.size(-1) : 0;
  if (x.is_cuda() && count > 0 && weight.dim() == 2 && weight.size(0) > 0 && one_launch(count, features, weight.size(0))) {
    const int32_t dtype = type_of(x.scalar_type(), "rows");
    const Rows r = rows_of(x, "rows");
    const Tensor& b = value_or_none(bias);
    const int64_t columns = weight.size(0), padded = padded_features(features);
    check_weight(weight, weight_scale, b, padded, columns, x.scalar_type());
    one_device(x, {&weight, &weight_scale, &b});
    const at::OptionalDeviceGuard guard(x.device());
    c10::SmallVector<int64_t, 3> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = columns;
    Tensor out = new_tensor(x, sizes, x.scalar_type());
    check(hb_int8_linear_rows(x.data_ptr(), r.batch_stride, r.row_stride, i32(r.batch, "batch"), i32(r.rows, "rows"),
                              i32(features, "features"), i32(columns, "columns"), i32(padded, "padded"), dtype, gelu,
                              static_cast<int8_t*>(weight.data_ptr()), static_cast<float*>(weight_scale.data_ptr()),
                              pointer(b), out.data_ptr(), r.rows * columns, columns, stream_of(x.device())),
          "hb_int8_linear_rows");
    return out;
  }
  const auto [q, scale] = int8_rows(x);
  return int8_linear(q, scale, weight, weight_scale, bias, x.scalar_type(), gelu);
}

void int8_linear_pair_out(const Tensor& q, const Tensor& scale, const Tensor& weight, const Tensor& weight_scale,
                      const Maybe& bias, Tensor out, const Tensor& q2, const Tensor& scale2, const Tensor& weight2,
                      const Tensor& weight_scale2, const Maybe& bias2, Tensor out2, bool gelu) {
  int8_linear_sets({{q, scale, weight, weight_scale, bias, out}, {q2, scale2, weight2, weight_scale2, bias2, out2}}, gelu);
}

// The text set's tensors are given together or not at all (its bias and norms may be missing).  An undefined `out` is
// made here, for `heads` heads in `type`.
void int8_qkv_into(const Maybe& text_q, const Maybe& text_scale, const Maybe& text_weight, const Maybe& text_weight_scale,
              const Maybe& text_bias, const Maybe& text_norm_q, const Maybe& text_norm_k, const Tensor& q,
              const Tensor& scale, const Tensor& weight, const Tensor& weight_scale, const Maybe& bias,
              const Maybe& norm_q, const Maybe& norm_k, const Maybe& cos, const Maybe& sin, Tensor& out, int64_t heads_of_new,
              at::ScalarType type, double eps) {
  if (!out.defined()) {
    type_of(type, "rows");
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) && q.size(1), "image must be nonempty [B, n, features] rows");
    TORCH_CHECK_VALUE(heads_of_new > 0, "heads must be positive");
    const Tensor& t = value_or_none(text_q);
    TORCH_CHECK_VALUE(!t.defined() || t.dim() == 3, "text must be [B, T, features] rows");
    out = new_tensor(q, {3, q.size(0), q.size(1) + (t.defined() ? t.size(1) : 0), heads_of_new, 128}, type);
  }
  TORCH_CHECK_VALUE(out.dim() == 5 && out.size(0) == 3 && out.size(3) > 0 && out.size(4) == 128,
                    "out must be [3, B, N, heads, 128]");
  const int32_t dtype = type_of(out.scalar_type(), "out");
  const int64_t batch = out.size(1), tokens = out.size(2), heads = out.size(3), columns = 3 * heads * 128;
  TORCH_CHECK_VALUE(out.stride(4) == 1 && (heads == 1 || out.stride(3) == 128), "out must have contiguous heads");
  const Tensor &tq = value_or_none(text_q), &ts = value_or_none(text_scale), &tw = value_or_none(text_weight),
               &tws = value_or_none(text_weight_scale), &co = value_or_none(cos), &si = value_or_none(sin);
  TORCH_CHECK_VALUE(tq.defined() == ts.defined() && tq.defined() == tw.defined() && tq.defined() == tws.defined(),
                    "text rows, their scales and their weight are given together");
  const int64_t padded = check_int8(q, scale, "image rows");
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == batch, "image rows must be [B, n, padded]");
  int64_t text = 0;
  void* pointers[14] = {};
  for (int part = tq.defined() ? 0 : 1; part < 2; ++part) {
    const Tensor &r = part ? q : tq, &rs = part ? scale : ts, &w = part ? weight : tw, &ws = part ? weight_scale : tws;
    const Tensor& b = value_or_none(part ? bias : text_bias);
    TORCH_CHECK_VALUE(check_int8(r, rs, "rows") == padded && r.dim() == 3 && r.size(0) == batch,
                      "text and image rows must be [B, rows, padded] of one batch and feature count");
    if (part == 0) text = r.size(1);
    check_weight(w, ws, b, padded, columns, out.scalar_type());
    void** p = pointers + 7 * part;
    void* values[5] = {pointer(r), pointer(rs), pointer(w), pointer(ws), pointer(b)};
    std::copy(values, values + 5, p);
    const Tensor& nq = value_or_none(part ? norm_q : text_norm_q);
    const Tensor& nk = value_or_none(part ? norm_k : text_norm_k);
    for (const Tensor* n : {&nq, &nk})
      TORCH_CHECK_VALUE(!n->defined() || (n->dim() == 1 && n->size(0) == 128 && n->is_contiguous() &&
                                          n->scalar_type() == out.scalar_type()),
                        "norm weights are contiguous [128] tensors of out's dtype");
    p[5] = pointer(nq);
    p[6] = pointer(nk);
    one_device(q, {&r, &rs, &w, &ws, &b, &nq, &nk});
    check_written(out, "out", {&r, &rs, &w, &ws, &b, &nq, &nk});
  }
  TORCH_CHECK_VALUE(text + q.size(1) == tokens, "out must hold the text rows and then the image rows");
  TORCH_CHECK_VALUE(co.defined() == si.defined(), "cos and sin must be given together");
  for (const Tensor* t : {&co, &si})
    TORCH_CHECK_VALUE(!t->defined() || (t->dim() == 2 && t->size(0) == tokens && t->size(1) == 128 &&
                                        t->is_contiguous() && t->scalar_type() == at::kFloat),
                      "cos/sin must be contiguous float32 [N, 128]");
  check_written(out, "out", {&co, &si});
  one_device(q, {&co, &si, &out});
  require_hip(q);
  const at::OptionalDeviceGuard guard(q.device());
  check(hb_int8_qkv(i32(batch, "batch"), i32(text, "text tokens"), i32(tokens, "tokens"), i32(heads, "heads"),
                    i32(padded, "padded"), dtype, static_cast<float>(eps), pointers, static_cast<float*>(pointer(co)),
                    static_cast<float*>(pointer(si)), out.data_ptr(), out.stride(0), batch == 1 ? 0 : out.stride(1),
                    tokens == 1 ? 0 : out.stride(2), stream_of(q.device())),
        "hb_int8_qkv");
}

void int8_qkv_out(const Maybe& text_q, const Maybe& text_scale, const Maybe& text_weight, const Maybe& text_weight_scale,
                  const Maybe& text_bias, const Maybe& text_norm_q, const Maybe& text_norm_k, const Tensor& q,
                  const Tensor& scale, const Tensor& weight, const Tensor& weight_scale, const Maybe& bias,
                  const Maybe& norm_q, const Maybe& norm_k, const Maybe& cos, const Maybe& sin, Tensor out, double eps) {
  int8_qkv_into(text_q, text_scale, text_weight, text_weight_scale, text_bias, text_norm_q, text_norm_k, q, scale, weight,
                weight_scale, bias, norm_q, norm_k, cos, sin, out, 0, out.scalar_type(), eps);
}

Tensor int8_qkv(const Maybe& text_q, const Maybe& text_scale, const Maybe& text_weight, const Maybe& text_weight_scale,
                const Maybe& text_bias, const Maybe& text_norm_q, const Maybe& text_norm_k, const Tensor& q,
                const Tensor& scale, const Tensor& weight, const Tensor& weight_scale, const Maybe& bias,
                const Maybe& norm_q, const Maybe& norm_k, const Maybe& cos, const Maybe& sin, at::ScalarType dtype,
                int64_t heads, double eps) {
  Tensor out;
  int8_qkv_into(text_q, text_scale, text_weight, text_weight_scale, text_bias, text_norm_q, text_norm_k, q, scale, weight,
                weight_scale, bias, norm_q, norm_k, cos, sin, out, heads, dtype, eps);
  return out;
}

// The attention operators and the 8-bit ones return nothing and write `out` and `lse` (and the like),
// which torch's own boxed fallbacks overlook: they look after returned tensors only.

// (the 8-bit operators that return their results write nothing)
constexpr const char* WRITING[] = {"paired_fwd", "sparse_fwd", "int8_adaln", "int8_adaln_pair", "int8_linear_out",
                                   "int8_linear_pair_out", "int8_qkv_out"};
constexpr const char* RETURNING[] = {"int8_rows", "int8_linear", "int8_linear_rows", "int8_qkv"};

// No derivative is recorded (the entry points refuse inputs that need one); a transform that takes one
// is refused, as torch refuses an autograd.Function in one, for it would get zeros.
void no_derivative(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const size_t count = op.schema().arguments().size();
  // (the attention operators' entry points look for gradients themselves; the 8-bit ones leave it to this)
  const bool refuse = at::GradMode::is_enabled() && op.schema().name().rfind("hilberta_hip::int8_", 0) == 0;
  // (included for as long as any torch.func transform is active)
  const bool transformed = at::GradMode::is_enabled() &&
                           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerBackMode);
  for (const c10::IValue& value : torch::jit::last(stack, count)) {
    if (!value.isTensor() || !value.toTensor().defined()) continue;
    const Tensor& t = value.toTensor();
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), "Trying to use forward AD with ",
                                op.schema().name(), " that does not support it.");
    TORCH_CHECK_VALUE(!(refuse && !transformed && t.requires_grad()), "Inference only; disable autograd");
    TORCH_CHECK(!(transformed && t.requires_grad()), op.schema().name(), " has no derivative for torch.func transforms");
  }
  const at::AutoDispatchBelowAutograd below;
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

// A tensor saved for a backward and then overwritten here has to fail that backward: every written
// argument's version counts up.
void counts_writes(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const auto& arguments = op.schema().arguments();
  const auto values = torch::jit::last(stack, arguments.size());
  c10::SmallVector<Tensor, 2> written;
  for (size_t i = 0; i < arguments.size(); ++i) {
    const c10::AliasInfo* alias = arguments[i].alias_info();
    if (alias && alias->isWrite() && values[i].isTensor() && values[i].toTensor().defined())
      written.push_back(values[i].toTensor());
  }
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
  }
  for (const Tensor& t : written)
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

}  // namespace

TORCH_LIBRARY(hilberta_hip, m) {
  const std::vector<at::Tag> tags{at::Tag::pt2_compliant_tag};
  m.def("paired_fwd(Tensor q, Tensor k, Tensor v, Tensor(a3!) out, Tensor(a4!)? lse, Tensor kv_indices, "
        "Tensor kv_flags, Tensor kv_counts, SymInt global_tokens, SymInt key_block_size, float scale_log2, "
        "bool all_queries, SymInt num_groups) -> ()", tags);
  m.def("sparse_fwd(Tensor q, Tensor k, Tensor v, Tensor(a3!) out, Tensor(a4!)? lse, Tensor kv_indices, "
        "Tensor kv_counts, SymInt global_tokens, float scale_log2, bool all_queries, SymInt num_groups) -> ()",
        tags);
  m.def("pair_rows(Tensor kv_indices, Tensor kv_counts, SymInt total_blocks, SymInt key_block_size, "
        "SymInt paired_width) -> (Tensor, Tensor, Tensor)", tags);
  m.def("gather_rows(Tensor x, SymInt dim, Tensor index) -> Tensor", tags);
  m.def("int8_rows(Tensor x) -> (Tensor, Tensor)", tags);
  const std::string ada = "Tensor x$, Tensor shift$, Tensor scale$, Tensor? y$, Tensor? gate$, Tensor(x$!)? x_out$, ",
                    linear = "Tensor q$, Tensor scale$, Tensor weight$, Tensor weight_scale$, Tensor? bias$, "
                             "Tensor(o$!) out$, ";
  const auto set = [](std::string text, const std::string& suffix) {
    for (size_t at; (at = text.find('$')) != std::string::npos;) text.replace(at, 1, suffix);
    return text;
  };
  m.def(("int8_adaln(" + set(ada, "") + "float eps) -> (Tensor, Tensor)").c_str(), tags);
  m.def(("int8_adaln_pair(" + set(ada, "") + set(ada, "2") + "float eps) -> (Tensor, Tensor, Tensor, Tensor)").c_str(), tags);
  m.def("int8_linear(Tensor q, Tensor scale, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType dtype, "
        "bool gelu) -> Tensor", tags);
  m.def("int8_linear_rows(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias, bool gelu) -> Tensor", tags);
  m.def(("int8_linear_out(" + set(linear, "") + "bool gelu) -> ()").c_str(), tags);
  m.def(("int8_linear_pair_out(" + set(linear, "") + set(linear, "2") + "bool gelu) -> ()").c_str(), tags);
  const std::string qkv = "Tensor? text_q, Tensor? text_scale, Tensor? text_weight, Tensor? text_weight_scale, "
                          "Tensor? text_bias, Tensor? text_norm_q, Tensor? text_norm_k, Tensor q, Tensor scale, Tensor weight, "
                          "Tensor weight_scale, Tensor? bias, Tensor? norm_q, Tensor? norm_k, Tensor? cos, Tensor? sin, ";
  m.def(("int8_qkv(" + qkv + "ScalarType dtype, SymInt heads, float eps) -> Tensor").c_str(), tags);
  m.def(("int8_qkv_out(" + qkv + "Tensor(a16!) out, float eps) -> ()").c_str(), tags);
  m.def("_attention_workspace(Device device, int need) -> Tensor");
  m.def("_workspace_keys() -> int[]");
  m.def("_clear_workspaces() -> ()");
  m.def("_abi_version() -> int");
}

TORCH_LIBRARY_IMPL(hilberta_hip, CUDA, m) {
  m.impl("paired_fwd", paired_fwd);
  m.impl("sparse_fwd", sparse_fwd);
  m.impl("pair_rows", pair_rows);
  m.impl("gather_rows", gather_rows);
}

// (on CPU tensors the 8-bit operators make their checks and refuse)
void int8_operators(torch::Library& m) {
  m.impl("int8_rows", int8_rows);
  m.impl("int8_adaln", int8_adaln);
  m.impl("int8_adaln_pair", int8_adaln_pair);
  m.impl("int8_linear", int8_linear);
  m.impl("int8_linear_rows", int8_linear_rows);
  m.impl("int8_linear_out", int8_linear_out);
  m.impl("int8_linear_pair_out", int8_linear_pair_out);
  m.impl("int8_qkv", int8_qkv);
  m.impl("int8_qkv_out", int8_qkv_out);
}
TORCH_LIBRARY_IMPL(hilberta_hip, CUDA, int8_hip) { int8_operators(int8_hip); }
TORCH_LIBRARY_IMPL(hilberta_hip, CPU, int8_cpu) { int8_operators(int8_cpu); }

TORCH_LIBRARY_IMPL(hilberta_hip, CompositeExplicitAutograd, m) {
  m.impl("_attention_workspace", attention_workspace);
  m.impl("_workspace_keys", workspace_keys);
  m.impl("_clear_workspaces", clear_workspaces);
  m.impl("_abi_version", abi_version);
}

// gather_rows and pair_rows: a differentiated call fails in its backward.
TORCH_LIBRARY_IMPL(hilberta_hip, Autograd, m) {
  for (const char* name : {"pair_rows", "gather_rows"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
  for (const char* name : WRITING)
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
  for (const char* name : RETURNING)
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
}

TORCH_LIBRARY_IMPL(hilberta_hip, ADInplaceOrView, m) {
  for (const char* name : WRITING)
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&counts_writes>());
}
