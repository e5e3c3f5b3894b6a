// Thin torch extension over the C ABI of libint8kv.so (include/int8kv.h): the drop-in operators
// int8_paged_attention, bf16_paged_attention and int8_kv_cache_write, and a serving step's
// build_batch_tables, lora_add and sample_tokens (serving_ops.h), called from Python
// with one pybind11 call each, instead of a Python wrapper plus a ctypes call of ~30 marshalled
// arguments.
//
// What it does per call, and nothing else: the reference's argument checks (raising the same
// exception types: AssertionError for the asserts of src/triton_ops/int8_paged_attention.py:
// 698-719 / int8_cache_write.py:100-115 / bf16_paged_attention.py:118-127, ValueError for an
// unknown impl, :767-768), the output and the decode workspace from torch's caching allocator on
// the input's device, torch's current HIP stream, and one C-ABI call whose strides are the
// tensors' own stride arrays.  No kernel lives here and no state is kept besides the exception
// class the library's status codes are raised as.

#include <torch/extension.h>

#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <map>
#include <string>
#include <utility>

#include "int8kv.h"
#include "serving_ops.h"

namespace {

namespace py = pybind11;

struct AssertionFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct ValueFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct LibraryFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

PyObject* g_library_error = PyExc_RuntimeError;  // int8kv._lib.Int8KVError once registered

inline void require(bool ok, const char* what = "") {
  if (!ok) throw AssertionFailure(what);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return INT8KV_F32;
    case at::kHalf: return INT8KV_F16;
    case at::kBFloat16: return INT8KV_BF16;
    case at::kChar: return INT8KV_I8;
    case at::kInt: return INT8KV_I32;
    case at::kLong: return INT8KV_I64;
    default: return -1;
  }
}

const char* status_text(int st) {
  switch (st) {
    case INT8KV_E_NULL: return "INT8KV_E_NULL (a required pointer is NULL)";
    case INT8KV_E_DTYPE: return "INT8KV_E_DTYPE (unsupported element type)";
    case INT8KV_E_SHAPE: return "INT8KV_E_SHAPE (unsupported or inconsistent size)";
    case INT8KV_E_STRIDE: return "INT8KV_E_STRIDE (innermost stride != 1 or rows not 16-byte aligned)";
    case INT8KV_E_WORKSPACE: return "INT8KV_E_WORKSPACE (workspace missing or too small)";
    case INT8KV_E_SCRATCH: return "INT8KV_E_SCRATCH (the call's split partials exceed the library's fixed scratch array)";
    default: return nullptr;
  }
}

void check_status(int st, const char* entry) {
  if (st == 0) return;
  const char* text = status_text(st);
  throw LibraryFailure(std::string(entry) + " failed: " +
                       (text ? std::string(text) : "hipError_t " + std::to_string(st)));
}

bool is_float_source(at::ScalarType t) {
  return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat;
}
bool is_index(at::ScalarType t) { return t == at::kInt || t == at::kLong; }

// 16-byte aligned base and row strides (dims) with a unit innermost stride.
bool rows_aligned16(const at::Tensor& t, std::initializer_list<int> dims) {
  const int64_t e = t.element_size();
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 || t.stride(-1) != 1) return false;
  for (int d : dims)
    if ((t.stride(d) * e) % 16) return false;
  return true;
}

// A contiguous copy at a fresh (aligned) address; .contiguous() would keep a misaligned offset.
at::Tensor fresh_copy(const at::Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }

at::Tensor fp32_vector(const at::Tensor& s) {
  return (s.scalar_type() == at::kFloat && s.is_contiguous()) ? s : s.to(at::kFloat).contiguous();
}

hipStream_t current_stream(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

constexpr int64_t kMaxRanges = 1 << 20;
constexpr int64_t kMaxSplits = 64;  // workgroups per (sequence, kv head) the split merge combines

// The reference's num_splits (src/triton_ops/int8_paged_attention.py:590-604) as the library's
// (num_ranges, flags): none = automatic; 1 = a single pass (one workgroup per sequence and kv
// head, INT8KV_DECODE_PER_SEQUENCE); S >= 2 = S workgroups per sequence and kv head over equal
// shares of its tiles (INT8KV_DECODE_SPLIT_SEQUENCES with num_ranges = S x batch), at most 64.
std::pair<int32_t, uint32_t> split_request(int64_t batch, const c10::optional<int64_t>& num_splits) {
  if (!num_splits.has_value()) return {0, 0u};
  if (*num_splits <= 1) return {0, INT8KV_DECODE_PER_SEQUENCE};
  const int64_t s = std::min<int64_t>(*num_splits, kMaxSplits);
  const int64_t r = std::min<int64_t>(kMaxRanges, s * std::max<int64_t>(1, batch));
  return {(int32_t)r, INT8KV_DECODE_SPLIT_SEQUENCES};
}

// Workspace of an eager call, kept per (device, stream) for the calling host thread: a call's
// partial records are read only by its own merge launch on the same stream, so the next call on
// that stream can reuse the buffer in stream order, while other streams and threads get their
// own.  Saves a caching-allocator round trip per call (~1.3 us of host time on MI355X).  Under
// graph capture it comes from torch's allocator instead (the graph's pool), so a replay never
// shares memory with eager calls.  The tensors are released when the thread ends.
at::Tensor workspace_for(const at::Tensor& like, hipStream_t stream, size_t need) {
  const int64_t bytes = (int64_t)std::max<size_t>(need, 16);
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone)
    return at::empty({bytes}, like.options().dtype(at::kByte));
  thread_local std::map<std::pair<int, uintptr_t>, at::Tensor> cache;
  at::Tensor& ws = cache[{(int)like.device().index(), reinterpret_cast<uintptr_t>(stream)}];
  if (!ws.defined() || ws.numel() < bytes) ws = at::empty({bytes}, like.options().dtype(at::kByte));
  return ws;
}

// Launches int8kv_paged_decode into `out`; the workspace comes from `workspace` when it is large
// enough, else from workspace_for.
at::Tensor decode_into(at::Tensor query, const at::Tensor& key_cache, const at::Tensor& value_cache,
                       const at::Tensor& block_tables, at::Tensor seq_lens,
                       const c10::optional<at::Tensor>& k_scale,
                       const c10::optional<at::Tensor>& v_scale, at::Tensor out, int64_t num_ranges,
                       int64_t flags, const c10::optional<at::Tensor>& workspace,
                       int64_t min_tiles) {
  const int64_t B = query.size(0), Hq = query.size(1), D = query.size(2);
  if (B == 0) return out;
  const int64_t NB = key_cache.size(0), BS = key_cache.size(1), Hkv = key_cache.size(2);
  if (!rows_aligned16(query, {0, 1})) query = fresh_copy(query);
  if (!seq_lens.is_contiguous()) seq_lens = seq_lens.contiguous();
  const size_t need = int8kv_decode_workspace_bytes((int32_t)Hq, (int32_t)Hkv, (int32_t)D,
                                                    (int32_t)BS, (int32_t)num_ranges);
  const hipStream_t stream = current_stream(query);
  const at::Tensor ws = (workspace.has_value() && (size_t)workspace->numel() >= need)
                            ? *workspace
                            : workspace_for(query, stream, need);
  const int st = int8kv_paged_decode(
      query.data_ptr(), dtype_code(query.scalar_type()), B, (int32_t)Hq, (int32_t)D,
      query.strides().data(), key_cache.data_ptr(), value_cache.data_ptr(),
      dtype_code(key_cache.scalar_type()), NB, (int32_t)BS, (int32_t)Hkv,
      key_cache.strides().data(), value_cache.strides().data(), block_tables.data_ptr(),
      dtype_code(block_tables.scalar_type()), block_tables.size(1), block_tables.strides().data(),
      seq_lens.data_ptr(), dtype_code(seq_lens.scalar_type()),
      k_scale.has_value() ? k_scale->data_ptr<float>() : nullptr,
      v_scale.has_value() ? v_scale->data_ptr<float>() : nullptr, (float)(1.0 / std::sqrt((double)D)),
      out.data_ptr(), out.strides().data(), ws.data_ptr(), (size_t)ws.numel(), (int32_t)num_ranges,
      (int32_t)min_tiles, (uint32_t)flags, stream);
  check_status(st, "int8kv_paged_decode");
  return out;
}

void require_same_device(std::initializer_list<const at::Tensor*> ts, const at::Tensor& first) {
  for (const at::Tensor* t : ts)
    require(t->device() == first.device(), "all tensors must be on one device (the GPU)");
}

// head_dims the decode kernels run (the reference pads any head_dim to a power of two under a
// mask, src/triton_ops/int8_paged_attention.py:556-558,588-589; other sizes fail here, before
// the C ABI, with the reference's AssertionError).
bool head_dim_ok(int64_t d) { return d >= 16 && d <= 256 && d % 16 == 0; }
const char* const kHeadDimText =
    "head_dim must be a multiple of 16 from 16 to 256 (this build's decode kernels)";

// src/triton_ops/int8_paged_attention.py:683-769 (validation :698-719, impl :767-768).
at::Tensor int8_paged_attention(const at::Tensor& query, const at::Tensor& key_cache,
                                const at::Tensor& value_cache, const at::Tensor& block_tables,
                                const at::Tensor& seq_lens, const at::Tensor& k_scale,
                                const at::Tensor& v_scale, bool quantize_q, const std::string& impl,
                                c10::optional<int64_t> num_splits) {
  require(query.dim() == 3 && key_cache.dim() == 4 && value_cache.dim() == 4);
  require(block_tables.dim() == 2 && seq_lens.dim() == 1);
  require(is_float_source(query.scalar_type()));
  require(key_cache.scalar_type() == at::kChar && value_cache.scalar_type() == at::kChar);
  require(is_index(block_tables.scalar_type()) && is_index(seq_lens.scalar_type()));
  const int64_t B = query.size(0), Hq = query.size(1), D = query.size(2);
  const int64_t Hkv = key_cache.size(2);
  require(value_cache.sizes() == key_cache.sizes());
  require(Hkv > 0, "key_cache has no kv heads");
  require(key_cache.size(3) == D && Hq % Hkv == 0);
  require(head_dim_ok(D), kHeadDimText);
  require(block_tables.size(0) == B && seq_lens.numel() == B);
  require(k_scale.dim() == 1 && v_scale.dim() == 1);
  require(k_scale.numel() == Hkv && v_scale.numel() == Hkv);
  require(key_cache.stride(-1) == 1 && value_cache.stride(-1) == 1);
  require(query.is_cuda(), "int8_paged_attention needs GPU tensors");
  require_same_device({&key_cache, &value_cache, &block_tables, &seq_lens, &k_scale, &v_scale},
                      query);
  if (impl != "auto" && impl != "v3" && impl != "v4")
    throw ValueFailure("Unknown impl='" + impl + "'; expected 'auto', 'v3' or 'v4'");
  if (impl == "v3" && !num_splits.has_value()) num_splits = 1;
  at::Tensor out = at::empty({B, Hq, D}, query.options());
  const auto split = split_request(B, num_splits);
  const int64_t flags =
      INT8KV_DECODE_ALL | split.second | (quantize_q ? INT8KV_DECODE_QUANTIZE_Q : 0);
  return decode_into(query, key_cache, value_cache, block_tables, seq_lens, fp32_vector(k_scale),
                     fp32_vector(v_scale), out, split.first, flags, c10::nullopt, 0);
}

// src/triton_ops/bf16_paged_attention.py:118-165.
at::Tensor bf16_paged_attention(const at::Tensor& query, const at::Tensor& key_cache,
                                const at::Tensor& value_cache, const at::Tensor& block_tables,
                                const at::Tensor& seq_lens, c10::optional<int64_t> num_splits) {
  require(query.dim() == 3 && key_cache.dim() == 4 && value_cache.dim() == 4);
  require(block_tables.dim() == 2 && seq_lens.dim() == 1);
  require(is_float_source(query.scalar_type()));
  require(key_cache.scalar_type() == at::kBFloat16 || key_cache.scalar_type() == at::kHalf);
  require(value_cache.scalar_type() == key_cache.scalar_type());
  require(is_index(block_tables.scalar_type()) && is_index(seq_lens.scalar_type()));
  const int64_t B = query.size(0), Hq = query.size(1), D = query.size(2);
  require(value_cache.sizes() == key_cache.sizes());
  require(key_cache.size(2) > 0, "key_cache has no kv heads");
  require(key_cache.size(3) == D && Hq % key_cache.size(2) == 0);
  require(head_dim_ok(D), kHeadDimText);
  require(block_tables.size(0) == B && seq_lens.numel() == B);
  require(key_cache.stride(-1) == 1 && value_cache.stride(-1) == 1);
  require(query.is_cuda(), "bf16_paged_attention needs GPU tensors");
  require_same_device({&key_cache, &value_cache, &block_tables, &seq_lens}, query);
  at::Tensor out = at::empty({B, Hq, D}, query.options());
  const auto split = split_request(B, num_splits);
  return decode_into(query, key_cache, value_cache, block_tables, seq_lens, c10::nullopt,
                     c10::nullopt, out, split.first, INT8KV_DECODE_ALL | split.second,
                     c10::nullopt, 0);
}

// src/triton_ops/int8_cache_write.py:85-149 (validation :100-115).
void int8_kv_cache_write(at::Tensor key, at::Tensor value, const at::Tensor& key_cache,
                         const at::Tensor& value_cache, at::Tensor slot_mapping,
                         const at::Tensor& k_scale, const at::Tensor& v_scale) {
  require(key.dim() == 3 && value.dim() == 3);
  require(key_cache.dim() == 4 && value_cache.dim() == 4);
  require(key.sizes() == value.sizes() && key_cache.sizes() == value_cache.sizes());
  require(key_cache.scalar_type() == at::kChar && value_cache.scalar_type() == at::kChar);
  require(is_float_source(key.scalar_type()) && is_float_source(value.scalar_type()));
  const int64_t T = key.size(0), Hkv = key.size(1), D = key.size(2);
  require(key_cache.size(2) == Hkv && key_cache.size(3) == D);
  require(slot_mapping.dim() == 1 && slot_mapping.numel() == T);
  require(k_scale.dim() == 1 && v_scale.dim() == 1);
  require(k_scale.numel() == Hkv && v_scale.numel() == Hkv);
  require(is_index(slot_mapping.scalar_type()));
  require(key.is_cuda(), "int8_kv_cache_write needs GPU tensors");
  require_same_device({&value, &key_cache, &value_cache, &slot_mapping, &k_scale, &v_scale}, key);
  require(key_cache.stride(-1) == 1 && value_cache.stride(-1) == 1);
  if (T == 0) return;
  if (value.scalar_type() != key.scalar_type()) {
    // One source type per launch; widening to fp32 is exact, so the quotients are unchanged.
    key = key.to(at::kFloat);
    value = value.to(at::kFloat);
  }
  if (!rows_aligned16(key, {0, 1})) key = fresh_copy(key);
  if (!rows_aligned16(value, {0, 1})) value = fresh_copy(value);
  if (!slot_mapping.is_contiguous()) slot_mapping = slot_mapping.contiguous();
  const at::Tensor ks = fp32_vector(k_scale), vs = fp32_vector(v_scale);
  const int st = int8kv_cache_write(
      key.data_ptr(), value.data_ptr(), dtype_code(key.scalar_type()), T, (int32_t)Hkv, (int32_t)D,
      key.strides().data(), value.strides().data(), key_cache.data_ptr(), value_cache.data_ptr(),
      key_cache.size(0), (int32_t)key_cache.size(1), key_cache.strides().data(),
      value_cache.strides().data(), slot_mapping.data_ptr(), dtype_code(slot_mapping.scalar_type()),
      ks.data_ptr<float>(), vs.data_ptr<float>(), current_stream(key));
  check_status(st, "int8kv_cache_write");
}

// The library's decode launcher with caller-chosen ranges/flags/workspace (the decode loop's
// per-layer call, the benchmark's kernel-only timing).
at::Tensor paged_decode(const at::Tensor& query, const at::Tensor& key_cache,
                        const at::Tensor& value_cache, const at::Tensor& block_tables,
                        const at::Tensor& seq_lens, const c10::optional<at::Tensor>& k_scale,
                        const c10::optional<at::Tensor>& v_scale, at::Tensor out, int64_t num_ranges,
                        int64_t flags, const c10::optional<at::Tensor>& workspace, int64_t min_tiles) {
  require(query.dim() == 3 && key_cache.dim() == 4 && value_cache.dim() == 4 &&
          out.sizes() == query.sizes());
  require(block_tables.dim() == 2 && seq_lens.dim() == 1);
  require(value_cache.sizes() == key_cache.sizes());
  require(query.is_cuda(), "paged_decode needs GPU tensors");
  require_same_device({&key_cache, &value_cache, &block_tables, &seq_lens, &out}, query);
  if (k_scale.has_value()) require(k_scale->device() == query.device() && k_scale->dim() == 1);
  if (v_scale.has_value()) require(v_scale->device() == query.device() && v_scale->dim() == 1);
  return decode_into(query, key_cache, value_cache, block_tables, seq_lens, k_scale, v_scale, out,
                     num_ranges, flags, workspace, min_tiles);
}

// int8kv/batch_tables.py (the same checks).
void build_batch_tables(at::Tensor computed_lens, at::Tensor new_lens, const at::Tensor& block_tables,
                        at::Tensor free_blocks, int64_t num_tokens, int64_t block_size,
                        const c10::optional<at::Tensor>& free_start, const at::Tensor& query_starts,
                        const at::Tensor& seq_lens, const at::Tensor& positions,
                        const at::Tensor& slot_mapping, const at::Tensor& token_requests,
                        const at::Tensor& free_end) {
  require(computed_lens.dim() == 1 && new_lens.sizes() == computed_lens.sizes());
  require(is_index(computed_lens.scalar_type()) &&
          new_lens.scalar_type() == computed_lens.scalar_type());
  const int64_t requests = computed_lens.numel();
  require(block_tables.dim() == 2 && block_tables.size(0) == requests);
  require(block_tables.scalar_type() == at::kInt);
  require(block_tables.stride(1) == 1 || block_tables.size(1) <= 1 || requests == 0);
  require(block_tables.stride(0) >= block_tables.size(1) || requests <= 1,
          "rows of block_tables overlap");
  require(free_blocks.dim() == 1 && free_blocks.scalar_type() == at::kInt);
  require(num_tokens >= 0 && num_tokens <= 0x7fffffff, "num_tokens must lie in [0, 2^31 - 1]");
  require(block_size >= 1 && block_size <= 65536, "block_size must lie in [1, 65536]");
  require(computed_lens.is_cuda(), "build_batch_tables needs GPU tensors");
  if (free_start.has_value()) {
    require(free_start->scalar_type() == at::kLong && free_start->numel() == 1);
    require_same_device({&*free_start}, computed_lens);
  }
  const auto buffer = [&](const at::Tensor& t, at::ScalarType type, int64_t n) {
    require(t.scalar_type() == type && t.is_contiguous() && t.numel() == n);
    require(requests == 0 || n == 0 || (t.data_ptr() != computed_lens.data_ptr() &&
                                        t.data_ptr() != new_lens.data_ptr()),
            "an output shares memory with the lengths");
  };
  buffer(query_starts, at::kInt, requests + 1);
  buffer(seq_lens, at::kInt, requests);
  buffer(positions, at::kLong, num_tokens);
  buffer(slot_mapping, at::kLong, num_tokens);
  buffer(token_requests, at::kInt, num_tokens);
  buffer(free_end, at::kLong, 1);
  require_same_device({&new_lens, &block_tables, &free_blocks, &query_starts, &seq_lens, &positions,
                       &slot_mapping, &token_requests, &free_end},
                      computed_lens);
  computed_lens = computed_lens.contiguous();
  new_lens = new_lens.contiguous();
  free_blocks = free_blocks.contiguous();
  const c10::hip::HIPGuard guard(computed_lens.device().index());
  const hipStream_t stream = current_stream(computed_lens);
  const at::Tensor ws =
      workspace_for(computed_lens, stream, int8kv_batch_tables_workspace_bytes(requests));
  const int st = int8kv_batch_tables(
      computed_lens.data_ptr(), new_lens.data_ptr(), dtype_code(computed_lens.scalar_type()),
      requests, block_tables.data_ptr<int32_t>(), block_tables.size(1), block_tables.stride(0),
      (int32_t)block_size, free_blocks.data_ptr<int32_t>(), free_blocks.numel(),
      free_start.has_value() ? free_start->data_ptr<int64_t>() : nullptr, num_tokens,
      query_starts.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), positions.data_ptr<int64_t>(),
      slot_mapping.data_ptr<int64_t>(), token_requests.data_ptr<int32_t>(),
      free_end.data_ptr<int64_t>(), ws.data_ptr(), (size_t)ws.numel(), stream);
  check_status(st, "int8kv_batch_tables");
}

// int8kv/lora.py (the same checks): fills `plan`, or a new buffer.
at::Tensor lora_plan(at::Tensor adapter_ids, int64_t num_adapters, c10::optional<at::Tensor> plan) {
  require(adapter_ids.dim() == 1 && is_index(adapter_ids.scalar_type()));
  require(num_adapters >= 1 && num_adapters <= 4096, "num_adapters must lie in [1, 4096]");
  require(adapter_ids.is_cuda(), "lora_plan needs GPU tensors");
  const int64_t tokens = adapter_ids.numel();
  require(tokens <= (1 << 24), "at most 2^24 tokens");
  adapter_ids = adapter_ids.contiguous();
  const c10::hip::HIPGuard guard(adapter_ids.device().index());
  if (!plan.has_value())
    plan = at::empty({(int64_t)int8kv_lora_plan_bytes(tokens, (int32_t)num_adapters)},
                     adapter_ids.options().dtype(at::kByte));
  require_same_device({&*plan}, adapter_ids);
  const int st = int8kv_lora_plan(adapter_ids.data_ptr(), dtype_code(adapter_ids.scalar_type()),
                                  tokens, (int32_t)num_adapters, plan->data_ptr(),
                                  (size_t)plan->numel(), current_stream(adapter_ids));
  check_status(st, "int8kv_lora_plan");
  return *plan;
}

at::Tensor lora_add(const at::Tensor& base, const at::Tensor& x, const at::Tensor& lora_a,
                    const at::Tensor& lora_b, const at::Tensor& plan, int64_t plan_tokens,
                    int64_t plan_adapters, c10::optional<at::Tensor> scales,
                    c10::optional<at::Tensor> out) {
  const auto matrix = [&](const at::Tensor& t, int64_t dim) {
    require(t.dim() == dim && t.scalar_type() == at::kBFloat16, "lora_add takes bf16 matrices");
    require(t.stride(-1) == 1, "lora_add takes matrices with a unit inner stride");
  };
  matrix(base, 2);
  matrix(x, 2);
  matrix(lora_a, 3);
  matrix(lora_b, 3);
  const int64_t tokens = x.size(0), k = x.size(1), n = base.size(1);
  const int64_t adapters = lora_a.size(0), rank = lora_a.size(1);
  require(base.size(0) == tokens && lora_a.size(2) == k);
  require(lora_b.size(0) == adapters && lora_b.size(1) == n && lora_b.size(2) == rank);
  require(k % 8 == 0 && n % 8 == 0 && rank % 8 == 0 && rank >= 8 && rank <= 128 && k > 0 && n > 0,
          "k, n and rank must be multiples of 8, rank at most 128");
  require(plan_tokens == tokens && plan_adapters == adapters, "a plan of other sizes");
  require(x.is_cuda(), "lora_add needs GPU tensors");
  if (scales.has_value()) {
    require(scales->scalar_type() == at::kFloat && scales->dim() == 1 && scales->numel() == adapters);
    require_same_device({&*scales}, x);
    scales = scales->contiguous();
  }
  if (!out.has_value()) out = at::empty({tokens, n}, base.options());
  require(out->sizes() == base.sizes() && out->scalar_type() == at::kBFloat16 && out->stride(1) == 1);
  require_same_device({&base, &lora_a, &lora_b, &plan, &*out}, x);
  const c10::hip::HIPGuard guard(x.device().index());
  const hipStream_t stream = current_stream(x);
  const at::Tensor ws = workspace_for(
      x, stream, int8kv_lora_workspace_bytes(tokens, (int32_t)adapters, k, (int32_t)rank));
  const int st = int8kv_lora_add(
      base.data_ptr(), base.stride(0), x.data_ptr(), tokens, k, x.stride(0), lora_a.data_ptr(),
      lora_a.strides().data(), lora_b.data_ptr(), lora_b.strides().data(), (int32_t)adapters,
      (int32_t)rank, n, scales.has_value() ? scales->data_ptr<float>() : nullptr, plan.data_ptr(),
      (size_t)plan.numel(), out->data_ptr(), out->stride(0), ws.data_ptr(), (size_t)ws.numel(),
      stream);
  check_status(st, "int8kv_lora_add");
  return *out;
}

// int8kv/sampling.py (the same checks).
at::Tensor sample_tokens(const at::Tensor& logits, const at::Tensor& uniforms,
                         const c10::optional<at::Tensor>& temperature,
                         const c10::optional<at::Tensor>& top_k,
                         const c10::optional<at::Tensor>& top_p,
                         const c10::optional<at::Tensor>& min_p, c10::optional<at::Tensor> out) {
  require(logits.dim() == 2 && is_float_source(logits.scalar_type()));
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  require(vocab >= 1 && vocab <= (1 << 21), "vocab must lie in [1, 2^21]");
  require(rows <= (1 << 16), "at most 2^16 rows");
  require(logits.stride(1) == 1 || vocab == 1);
  require(logits.stride(0) >= vocab || rows <= 1, "rows of logits overlap");
  require(logits.is_cuda(), "sample_tokens needs GPU tensors");
  const auto setting = [&](const c10::optional<at::Tensor>& t, at::ScalarType type) {
    if (!t.has_value()) return at::Tensor();
    require(t->scalar_type() == type && t->dim() == 1 && t->numel() == rows);
    require_same_device({&*t}, logits);
    return t->contiguous();
  };
  const at::Tensor u = setting(uniforms, at::kFloat), te = setting(temperature, at::kFloat),
                   tk = setting(top_k, at::kInt), tp = setting(top_p, at::kFloat),
                   mp = setting(min_p, at::kFloat);
  if (!out.has_value()) out = at::empty({rows}, logits.options().dtype(at::kLong));
  require(out->scalar_type() == at::kLong && out->is_contiguous() && out->dim() == 1 &&
          out->numel() == rows);
  require_same_device({&*out}, logits);
  const c10::hip::HIPGuard guard(logits.device().index());
  const hipStream_t stream = current_stream(logits);
  const at::Tensor ws = workspace_for(logits, stream, int8kv_sample_workspace_bytes(rows, vocab));
  const auto f32 = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  const int st = int8kv_sample_rows(
      logits.data_ptr(), dtype_code(logits.scalar_type()), rows, vocab,
      std::max<int64_t>(logits.stride(0), vocab), f32(u), f32(te),
      tk.defined() ? tk.data_ptr<int32_t>() : nullptr, f32(tp), f32(mp), out->data_ptr<int64_t>(),
      ws.data_ptr(), (size_t)ws.numel(), stream);
  check_status(st, "int8kv_sample_rows");
  return *out;
}

void set_library_error(py::object cls) {
  cls.inc_ref();  // kept for the life of the process
  g_library_error = cls.ptr();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const AssertionFailure& e) {
      PyErr_SetString(PyExc_AssertionError, e.what());
    } catch (const ValueFailure& e) {
      PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const LibraryFailure& e) {
      PyErr_SetString(g_library_error, e.what());
    }
  });
  m.def("int8_paged_attention", &int8_paged_attention, py::arg("query"), py::arg("key_cache"),
        py::arg("value_cache"), py::arg("block_tables"), py::arg("seq_lens"), py::arg("k_scale"),
        py::arg("v_scale"), py::arg("quantize_q"), py::arg("impl"), py::arg("num_splits"));
  m.def("bf16_paged_attention", &bf16_paged_attention, py::arg("query"), py::arg("key_cache"),
        py::arg("value_cache"), py::arg("block_tables"), py::arg("seq_lens"), py::arg("num_splits"));
  m.def("int8_kv_cache_write", &int8_kv_cache_write, py::arg("key"), py::arg("value"),
        py::arg("key_cache"), py::arg("value_cache"), py::arg("slot_mapping"), py::arg("k_scale"),
        py::arg("v_scale"));
  m.def("paged_decode", &paged_decode, py::arg("query"), py::arg("key_cache"),
        py::arg("value_cache"), py::arg("block_tables"), py::arg("seq_lens"), py::arg("k_scale"),
        py::arg("v_scale"), py::arg("out"), py::arg("num_ranges"), py::arg("flags"),
        py::arg("workspace"), py::arg("min_tiles"));
  m.def("build_batch_tables", &build_batch_tables);
  m.def("lora_plan", &lora_plan);
  m.def("lora_add", &lora_add);
  m.def("sample_tokens", &sample_tokens);
  m.def("set_library_error", &set_library_error);
}
