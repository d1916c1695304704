// The batched-serving entry points as torch calls (gds_io_ext): argument
// checks, output allocation and the C ABI, in one crossing from Python.  The
// public functions are gdsllm_b200/paged.py and gdsllm_b200/sampling.py.
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "gdsq.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

// GdsqError (gdsllm_b200/_native.py) with the library's error text.
void check(int status, const char* what) {
  if (status == GDSQ_OK) return;
  const std::string text = std::string(what) + ": " + gdsq_status_string(status) + " (" + gdsq_last_error() + ")";
  py::object type = py::module_::import("gdsllm_b200._native").attr("GdsqError");
  PyErr_SetString(type.ptr(), text.c_str());
  throw py::error_already_set();
}

int elem_type(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return GDSQ_ELEM_F16;
    case at::kBFloat16: return GDSQ_ELEM_BF16;
    case at::kFloat: return GDSQ_ELEM_F32;
    default: return -1;
  }
}

const void* array(const Tensor& t, const char* name, int64_t n, const Tensor& like, at::ScalarType type = at::kInt) {
  NEED(t.scalar_type() == type && t.numel() == n && t.is_contiguous() && t.device() == like.device(), name, ": expected ", n,
       " contiguous ", type, " on ", like.device(), ", got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
  return t.const_data_ptr();
}
void* array_out(const Tensor& t, const char* name, int64_t n, const Tensor& like, at::ScalarType type = at::kInt) {
  return const_cast<void*>(array(t, name, n, like, type));
}

Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// A contiguous tensor `at` bytes into buffer's storage: several outputs of one call share one allocation.
Tensor part(const Tensor& buffer, int64_t at, at::IntArrayRef sizes, at::ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(),
                                                     c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(type)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

void on_gpu(const Tensor& t) { NEED(t.is_cuda(), "the tensors must be on a CUDA device, not ", t.device()); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int32_t small(int64_t n, const char* name) {
  NEED(n >= 0 && n <= INT32_MAX, name, " = ", n, " is not within 0 .. 2^31 - 1");
  return static_cast<int32_t>(n);
}

// A layer's cache, checked.
struct Cache {
  int type, blocks, heads, block, dim;
  Cache(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
    type = k.scalar_type() == at::kChar ? GDSQ_CACHE_INT8 : GDSQ_CACHE_E4M3;
    NEED(k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn, "the cache is int8 or float8_e4m3fn, not ",
         k.scalar_type());
    NEED(k.dim() == 4, "the cache is [blocks, kv_heads, block_size, dim], not ", k.sizes());
    NEED(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && k.is_contiguous() && v.is_contiguous() &&
             v.device() == k.device(), "k_cache and v_cache must be contiguous and alike");
    for (const Tensor* s : {&ks, &vs})
      NEED(s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == k.size(0) && s->size(1) == k.size(1) &&
               s->is_contiguous() && s->device() == k.device(), "the scales are contiguous fp32 [", k.size(0), ", ", k.size(1),
           "], got ", s->sizes(), " ", s->scalar_type());
    blocks = small(k.size(0), "blocks");
    heads = small(k.size(1), "kv_heads");
    block = small(k.size(2), "block_size");
    dim = small(k.size(3), "dim");
  }
};

// [tokens, heads, dim] activations with a contiguous last dimension.
void rows(const Tensor& x, const char* name, int64_t heads, int dim, const Tensor& like, const Tensor* type = nullptr) {
  NEED(x.dim() == 3 && x.size(2) == dim && (heads < 0 || x.size(1) == heads) && x.stride(2) == 1, name,
       ": expected [tokens, heads, ", dim, "] with unit stride, got ", x.sizes(), " strides ", x.strides());
  NEED((x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16) && x.device() == like.device() &&
           (!type || x.scalar_type() == type->scalar_type()), name, ": fp16 or bf16 on ", like.device(), ", all alike; got ",
       x.scalar_type(), " on ", x.device());
}

using Tables = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Tables build_tables(const Tensor& context, const Tensor& fresh, const Tensor& table, const Tensor& free_blocks,
                    const Tensor& free_head, int64_t block_size, int64_t num_tokens, const std::optional<Tables>& out) {
  const int64_t r = context.numel();
  NEED(table.dim() == 2 && table.size(0) == r, "block_table ", table.sizes(), " has not ", r, " rows");
  const void* c = array(context, "context_lens", r, context);
  const void* n = array(fresh, "new_lens", r, context);
  void* t = array_out(table, "block_table", r * table.size(1), context);
  const void* f = array(free_blocks, "free_blocks", free_blocks.numel(), context);
  const void* h = array(free_head, "free_head", 1, context);
  const int tokens = small(num_tokens, "num_tokens");
  on_gpu(context);
  const c10::cuda::CUDAGuard guard(context.device());
  Tables o;
  if (out) {
    o = *out;
  } else {
    const Tensor b = make({16 * num_tokens + 8 * (r + 1)}, at::kByte, context);
    const int64_t ints = 16 * num_tokens;
    o = Tables(part(b, ints, {r}, at::kInt), part(b, ints + 4 * r, {r + 1}, at::kInt), part(b, 0, {num_tokens}, at::kLong),
               part(b, 8 * num_tokens, {num_tokens}, at::kLong), part(b, ints + 8 * r + 4, {1}, at::kInt));
  }
  check(gdsq_build_tables(static_cast<const int32_t*>(c), static_cast<const int32_t*>(n), small(r, "requests"),
                          static_cast<int32_t*>(t), small(table.size(1), "table width"), static_cast<const int32_t*>(f),
                          small(free_blocks.numel(), "free blocks"), static_cast<const int32_t*>(h),
                          small(block_size, "block_size"), tokens,
                          static_cast<int32_t*>(array_out(std::get<0>(o), "out.seq_lens", r, context)),
                          static_cast<int32_t*>(array_out(std::get<1>(o), "out.query_starts", r + 1, context)),
                          static_cast<long long*>(array_out(std::get<2>(o), "out.positions", tokens, context, at::kLong)),
                          static_cast<long long*>(array_out(std::get<3>(o), "out.slots", tokens, context, at::kLong)),
                          static_cast<int32_t*>(array_out(std::get<4>(o), "out.free_head", 1, context)), stream_of(context)),
        "gdsq_build_tables");
  return o;
}

OptTensor append_kv8(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache,
                     const Tensor& k_scale, const Tensor& v_scale, const OptTensor& q, const OptTensor& freqs,
                     const OptTensor& positions, OptTensor q_out) {
  const Cache c(k_cache, v_cache, k_scale, v_scale);
  rows(k, "k", c.heads, c.dim, k_cache);
  rows(v, "v", c.heads, c.dim, k_cache, &k);
  const int64_t tokens = k.size(0);
  NEED(v.size(0) == tokens, "k has ", tokens, " tokens, v ", v.size(0));
  const void* sl = array(slots, "slots", tokens, k_cache, at::kLong);
  const void *fp = nullptr, *pp = nullptr, *qp = nullptr;
  int64_t limit = 0, qt = 0, qh = 0, heads = 0;
  if (freqs) {
    NEED(positions.has_value(), "freqs needs positions");
    NEED(freqs->scalar_type() == at::kFloat && freqs->dim() == 3 && freqs->size(1) == c.dim / 2 && freqs->size(2) == 2 &&
             freqs->is_contiguous() && freqs->device() == k_cache.device(), "freqs: contiguous fp32 [positions, ", c.dim / 2,
         ", 2] on ", k_cache.device(), ", got ", freqs->sizes(), " ", freqs->scalar_type());
    limit = freqs->size(0);
    fp = freqs->const_data_ptr();
    pp = array(*positions, "positions", tokens, k_cache, at::kLong);
  }
  if (q) {
    NEED(freqs.has_value(), "q is only rotated, which needs freqs");
    rows(*q, "q", -1, c.dim, k_cache, &k);
    NEED(q->size(0) == tokens, "k has ", tokens, " tokens, q ", q->size(0));
    heads = q->size(1);
    qp = q->const_data_ptr();
    qt = q->stride(0);
    qh = q->stride(1);
    if (q_out) {
      NEED(q_out->sizes() == q->sizes() && q_out->scalar_type() == q->scalar_type() && q_out->is_contiguous() &&
               q_out->device() == q->device(), "q_out: contiguous and like q");
    }
  }
  on_gpu(k_cache);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  if (q && !q_out) q_out = make(q->sizes(), q->scalar_type(), *q);
  check(gdsq_append_kv8(elem_type(k), qp, qt, qh, k.const_data_ptr(), k.stride(0), k.stride(1), v.const_data_ptr(), v.stride(0),
                        v.stride(1), q ? q_out->data_ptr() : nullptr, fp, small(limit, "freqs"),
                        static_cast<const long long*>(pp), static_cast<const long long*>(sl), small(tokens, "tokens"),
                        small(heads, "heads"), c.heads, c.dim, c.type, k_cache.data_ptr(), v_cache.data_ptr(),
                        k_scale.data_ptr<float>(), v_scale.data_ptr<float>(), c.blocks, c.block, stream_of(k_cache)),
        "gdsq_append_kv8");
  return q ? q_out : std::nullopt;
}

Tensor attend_workspace(int64_t requests, int64_t max_query_len, int64_t heads, int64_t kv_heads, int64_t dim, at::Device device) {
  NEED(device.is_cuda(), "attend_workspace: a CUDA device, not ", device);
  const c10::cuda::CUDAGuard guard(device);
  const size_t n = gdsq_attend_kv8_workspace(small(requests, "requests"), small(max_query_len, "max_query_len"),
                                             small(heads, "heads"), small(kv_heads, "kv_heads"), small(dim, "dim"));
  return at::zeros({static_cast<int64_t>(std::max<size_t>(n, 16))}, at::TensorOptions(at::kByte).device(device));
}

Tensor attend_kv8(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                  const Tensor& table, const Tensor& seq_lens, const Tensor& starts, int64_t max_query_len,
                  std::optional<int64_t> max_seq_len, std::optional<double> scale, OptTensor out, OptTensor workspace) {
  const Cache c(k_cache, v_cache, k_scale, v_scale);
  rows(q, "q", -1, c.dim, k_cache);
  const int64_t r = seq_lens.numel(), heads = q.size(1);
  NEED(table.dim() == 2 && table.size(0) == r, "block_table ", table.sizes(), " has not ", r, " rows");
  if (out) {
    NEED(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->is_contiguous() && out->device() == q.device(),
         "out: contiguous and like q");
  }
  if (workspace) NEED(workspace->device() == q.device() && workspace->is_contiguous(), "workspace: contiguous on ", q.device());
  const void* tb = array(table, "block_table", r * table.size(1), k_cache);
  const void* ln = array(seq_lens, "seq_lens", r, k_cache);
  const void* st = array(starts, "query_starts", r + 1, k_cache);
  on_gpu(q);
  const c10::cuda::CUDAGuard guard(q.device());
  if (!out) out = make(q.sizes(), q.scalar_type(), q);
  if (r == 0 || max_query_len == 0) out->zero_();  // no token belongs to a request; the C call has nothing to do
  if (!workspace) workspace = attend_workspace(r, max_query_len, heads, c.heads, c.dim, q.device());
  const int width = small(table.size(1), "table width");
  check(gdsq_attend_kv8(q.const_data_ptr(), elem_type(q), q.stride(0), q.stride(1), k_cache.const_data_ptr(),
                        v_cache.const_data_ptr(), c.type, k_scale.const_data_ptr<float>(), v_scale.const_data_ptr<float>(),
                        c.blocks, c.block, static_cast<const int32_t*>(tb), width, static_cast<const int32_t*>(ln),
                        static_cast<const int32_t*>(st), small(r, "requests"), small(q.size(0), "tokens"),
                        small(max_query_len, "max_query_len"),
                        small(max_seq_len.value_or(0), "max_seq_len"),
                        small(heads, "heads"), c.heads, c.dim,
                        static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(c.dim))), out->data_ptr(),
                        workspace->data_ptr(), workspace->nbytes(), stream_of(q)),
        "gdsq_attend_kv8");
  return *out;
}

std::tuple<Tensor, Tensor> sample(const Tensor& logits, const Tensor& uniforms, const OptTensor& temperature,
                                  const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p, OptTensor tokens,
                                  OptTensor logprobs) {
  NEED(logits.dim() == 2 && elem_type(logits) >= 0 && (logits.size(1) <= 1 || logits.stride(1) == 1),
       "logits: [rows, vocab] fp16, bf16 or fp32 with contiguous rows, got ", logits.sizes(), " ", logits.scalar_type(),
       " strides ", logits.strides());
  const int64_t b = logits.size(0);
  auto param = [&](const OptTensor& t, const char* name, at::ScalarType type) {
    return t ? array(*t, name, b, logits, type) : nullptr;
  };
  const void* u = array(uniforms, "uniforms", b, logits, at::kFloat);
  const void* t = param(temperature, "temperature", at::kFloat);
  const void* k = param(top_k, "top_k", at::kInt);
  const void* p = param(top_p, "top_p", at::kFloat);
  const void* m = param(min_p, "min_p", at::kFloat);
  param(tokens, "tokens", at::kLong);
  param(logprobs, "logprobs", at::kFloat);
  on_gpu(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  if (!tokens || !logprobs) {
    const Tensor both = make({12 * b}, at::kByte, logits);
    if (!tokens) tokens = part(both, 0, {b}, at::kLong);
    if (!logprobs) logprobs = part(both, 8 * b, {b}, at::kFloat);
  }
  check(gdsq_sample(elem_type(logits), logits.const_data_ptr(), logits.stride(0), small(b, "rows"),
                    small(logits.size(1), "vocab"), static_cast<const float*>(u), static_cast<const float*>(t),
                    static_cast<const int32_t*>(k), static_cast<const float*>(p), static_cast<const float*>(m),
                    static_cast<long long*>(tokens->data_ptr()), logprobs->data_ptr<float>(), stream_of(logits)),
        "gdsq_sample");
  return {*tokens, *logprobs};
}

}  // namespace

void bind_serving(py::module_& m) {
  m.def("build_tables", &build_tables, "A step's block table, positions and cache slots (gdsllm_b200.paged).");
  m.def("append_kv8", &append_kv8, "K and V into the 8-bit paged cache, with RoPE (gdsllm_b200.paged).");
  m.def("attend_workspace", [](int64_t r, int64_t n, int64_t h, int64_t kh, int64_t d, const py::object& device) {
    return attend_workspace(r, n, h, kh, d, at::Device(py::str(device).cast<std::string>()));
  }, "A zeroed workspace for attend_kv8 (gdsllm_b200.paged).");
  m.def("attend_kv8", &attend_kv8, "Attention over the 8-bit paged cache (gdsllm_b200.paged).");
  m.def("sample", &sample, "Tokens from logits and uniform numbers (gdsllm_b200.sampling).");
}
