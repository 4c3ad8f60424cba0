// PyTorch binding of libserving_ops.so (include/serving_ops.h): argument checks, results through the caching
// allocator, torch's current stream, a device guard.  No kernel here, nothing is kept between calls, nothing is
// synchronised: every call may be captured in a graph.  ValueError for shapes, RuntimeError for types and devices, as
// the AWQ operators have it.
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/serving_ops.h"

namespace {

using c10::hip::getCurrentHIPStreamMasqueradingAsCUDA;
using c10::hip::OptionalHIPGuardMasqueradingAsCUDA;
using torch::Tensor;

constexpr int64_t kMostInt = 0x7fffffff;

void raise_for(int rc, const char* what) {
  if (rc == SERVING_OK) return;
  const std::string msg = std::string(what) + ": " + serving_strerror(rc);
  switch (rc) {
    case SERVING_E_SHAPE:
    case SERVING_E_HEAD:
    case SERVING_E_BLOCK:
    case SERVING_E_ROTARY:
    case SERVING_E_TOO_LARGE:
      throw std::invalid_argument(msg);
    default:
      TORCH_CHECK(false, msg, rc == SERVING_E_LAUNCH ? " (hipError " + std::to_string(serving_last_hip_error()) + ")" : "");
  }
}

// The message is put together only where it is needed.
#define NEED(ok, ...)                                                          \
  do {                                                                         \
    if (!(ok)) throw std::invalid_argument(c10::str(what, ": ", __VA_ARGS__)); \
  } while (0)

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

void typed(const Tensor& t, at::ScalarType type, const char* what, const char* name) {
  TORCH_CHECK(t.scalar_type() == type, what, ": expected scalar type ", type, " but found ", t.scalar_type(), " for ", name);
}

// Half or BFloat16: whether it is BFloat16.
bool activations(const Tensor& t, const char* what, const char* name) {
  const auto type = t.scalar_type();
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, what, ": expected scalar type Half or BFloat16 but found ", type,
              " for ", name);
  return type == at::kBFloat16;
}

void on_gpu(const Tensor& t, const Tensor& like, const char* what, const char* name) {
  TORCH_CHECK(t.is_cuda(), what, ": ", name, " must be a GPU tensor: there is no CPU implementation");
  TORCH_CHECK(t.device() == like.device(), what, ": ", name, " is on another device than the rest");
}

void no_gradient(const Tensor& t, const char* what, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, ": ", name,
              " requires a gradient, which this operator does not give: call it under torch.no_grad() or on a detached tensor");
  TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()), what, ": ", name,
              " carries a tangent of forward-mode differentiation, which this operator does not pass on");
}

// What a call writes into counts as changed in place for whoever saved it for a backward pass.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Rows of heads whose elements lie together, at addresses and strides that 16-byte loads can take.
Tensor heads_of(const Tensor& t) {
  const bool fits = t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

Tensor ints(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

// D and P of a cache [blocks, kv heads, P (D + 8)] for heads of head_size elements.
int64_t block_size_of(const Tensor& cache, int64_t head_size, const char* what) {
  typed(cache, at::kByte, what, "cache");
  NEED(head_size == 64 || head_size == 128, "head_size must be 64 or 128, got ", head_size);
  NEED(cache.dim() == 3 && cache.size(0) > 0 && cache.size(1) > 0 && cache.size(2) > 0 && cache.size(2) % (head_size + 8) == 0 &&
           (cache.size(2) / (head_size + 8)) % 16 == 0, "cache must be [blocks, kv heads, block_size * (head_size + 8)] with a block_size that is a multiple of 16, got ", shape_of(cache), " for heads of ", head_size);
  NEED(cache.is_contiguous(), "cache must be contiguous");
  NEED(cache.size(0) <= kMostInt && cache.size(1) <= 65535 && cache.size(2) / (head_size + 8) <= 4096, "cache is too large");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0, what, ": cache is not 16-byte aligned");
  return cache.size(2) / (head_size + 8);
}

Tensor rope_append_kv4(const Tensor& positions, const Tensor& query, const Tensor& key, const Tensor& value,
                       const Tensor& cos_sin, const Tensor& cache, const Tensor& slots, bool interleaved) {
  const char* what = "rope_append_kv4";
  const bool bf16 = activations(query, what, "query");
  typed(key, query.scalar_type(), what, "key");
  typed(value, query.scalar_type(), what, "value");
  typed(cos_sin, at::kFloat, what, "cos_sin");
  typed(positions, at::kLong, what, "positions");
  typed(slots, at::kLong, what, "slots");
  NEED(query.dim() == 3, "query must be [tokens, heads, head_size], got ", shape_of(query));
  const int64_t tokens = query.size(0), heads = query.size(1), d = query.size(2);
  const int64_t block_size = block_size_of(cache, d, what), kv = cache.size(1);
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(key, "key"), {value, "value"}})
    NEED(t.dim() == 3 && t.size(0) == tokens && t.size(1) == kv && t.size(2) == d, name, " must be [", tokens, ", ", kv, ", ", d, "] as query and cache have it, got ", shape_of(t));
  NEED(positions.dim() == 1 && positions.size(0) == tokens, "positions must be [tokens], got ", shape_of(positions));
  NEED(slots.dim() == 1 && slots.size(0) == tokens, "slots must be [tokens], got ", shape_of(slots));
  NEED(cos_sin.dim() == 2, "cos_sin must be [positions, rotary], got ", shape_of(cos_sin));
  const int64_t rotary = cos_sin.size(1);
  NEED(rotary % 16 == 0 && rotary <= d, "the rotated part of a head must be a multiple of 16 elements and no larger than a head, got ", rotary);
  NEED(rotary == 0 || cos_sin.size(0) > 0, "cos_sin has no positions");
  NEED(tokens <= (1 << 30) && heads > 0 && heads <= 65535, "query has too many tokens, or ", heads, " heads");
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(query, "query"), {key, "key"}, {value, "value"},
                                {cos_sin, "cos_sin"}, {cache, "cache"}, {positions, "positions"}, {slots, "slots"}}) {
    on_gpu(t, query, what, name);
    no_gradient(t, what, name);
  }
  const OptionalHIPGuardMasqueradingAsCUDA guard(query.device());
  Tensor out = torch::empty({tokens, heads, d}, query.options());
  if (tokens == 0) return out;
  const Tensor q = heads_of(query), k = heads_of(key), v = heads_of(value), at = ints(positions), to = ints(slots);
  const bool table_fits = rotary == 0 || (cos_sin.stride(1) == 1 && cos_sin.stride(0) % 4 == 0 &&
                                          reinterpret_cast<uintptr_t>(cos_sin.data_ptr()) % 16 == 0);
  const Tensor cs = table_fits ? cos_sin : cos_sin.clone(at::MemoryFormat::Contiguous);
  raise_for(serving_rope_append_kv4(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                                    v.data_ptr(), v.stride(0), v.stride(1), rotary ? cs.data_ptr<float>() : nullptr,
                                    rotary ? cs.stride(0) : 0, at.data_ptr<int64_t>(), to.data_ptr<int64_t>(), out.data_ptr(),
                                    cache.data_ptr(), (int)tokens, (int)heads, (int)kv, (int)d, (int)rotary, interleaved,
                                    cos_sin.size(0), cache.size(0), (int)block_size, bf16,
                                    getCurrentHIPStreamMasqueradingAsCUDA().stream()),
            what);
  written(cache);
  return out;
}

std::tuple<Tensor, Tensor> kv4_read(const Tensor& cache, const Tensor& slots, int64_t head_size, at::ScalarType dtype) {
  const char* what = "kv4_read";
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, what, ": dtype must be Half or BFloat16, got ", dtype);
  const int64_t block_size = block_size_of(cache, head_size, what);
  typed(slots, at::kLong, what, "slots");
  NEED(slots.dim() == 1, "slots must be [rows], got ", shape_of(slots));
  on_gpu(cache, cache, what, "cache");
  on_gpu(slots, cache, what, "slots");
  const OptionalHIPGuardMasqueradingAsCUDA guard(cache.device());
  const int64_t rows = slots.size(0), kv = cache.size(1);
  Tensor key = torch::empty({rows, kv, head_size}, cache.options().dtype(dtype)), value = torch::empty_like(key);
  if (rows == 0) return {key, value};
  const Tensor from = ints(slots);
  raise_for(serving_read_kv4(cache.data_ptr(), from.data_ptr<int64_t>(), key.data_ptr(), value.data_ptr(), rows, (int)kv,
                             (int)head_size, cache.size(0), (int)block_size, dtype == at::kBFloat16,
                             getCurrentHIPStreamMasqueradingAsCUDA().stream()),
            what);
  return {key, value};
}

Tensor paged_attention_kv4(const Tensor& query, const Tensor& cache, const Tensor& block_tables, const Tensor& seq_lens,
                           double scale, int64_t max_seq_len, const std::optional<Tensor>& query_start, int64_t max_query_len,
                           int64_t window, const std::optional<Tensor>& out_) {
  const char* what = "paged_attention_kv4";
  const bool bf16 = activations(query, what, "query");
  typed(block_tables, at::kInt, what, "block_tables");
  typed(seq_lens, at::kInt, what, "seq_lens");
  NEED(query.dim() == 3, "query must be [tokens, heads, head_size], got ", shape_of(query));
  const int64_t tokens = query.size(0), heads = query.size(1), d = query.size(2);
  const int64_t block_size = block_size_of(cache, d, what), kv = cache.size(1);
  NEED(heads > 0 && heads <= 65535 && heads % kv == 0, "query has ", heads, " heads, which the cache's ", kv, " cannot share");
  NEED(seq_lens.dim() == 1, "seq_lens must be [sequences], got ", shape_of(seq_lens));
  const int64_t seqs = seq_lens.size(0);
  NEED(block_tables.dim() == 2 && block_tables.size(0) == seqs, "block_tables must be [sequences, blocks], got ", shape_of(block_tables));
  NEED(max_seq_len > 0 && max_seq_len <= (1 << 27) && block_tables.size(1) * block_size <= (1 << 27), "sequences are of 1 to 2^27 tokens");
  NEED(window >= 0 && window <= kMostInt, "window must not be negative");
  NEED(max_query_len > 0 && max_query_len <= kMostInt, "max_query_len must be positive");
  NEED(std::isfinite(scale) && std::isfinite((float)scale), "scale must be finite");
  NEED(tokens <= kMostInt, "too many tokens");
  if (query_start) {
    typed(*query_start, at::kInt, what, "query_start");
    NEED(query_start->dim() == 1 && query_start->size(0) == seqs + 1, "query_start must be [sequences + 1], got ", shape_of(*query_start));
    on_gpu(*query_start, query, what, "query_start");
  } else {
    NEED(tokens == seqs, "without query_start there is one query for each sequence");
    NEED(max_query_len == 1, "without query_start max_query_len is 1");
  }
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(query, "query"), {cache, "cache"},
                                {block_tables, "block_tables"}, {seq_lens, "seq_lens"}})
    on_gpu(t, query, what, name);
  no_gradient(query, what, "query");
  if (out_) {
    typed(*out_, query.scalar_type(), what, "out");
    on_gpu(*out_, query, what, "out");
    no_gradient(*out_, what, "out");
    NEED(out_->sizes() == query.sizes() && out_->is_contiguous(), "out must be a contiguous ", shape_of(query), ", got ", shape_of(*out_));
    TORCH_CHECK(reinterpret_cast<uintptr_t>(out_->data_ptr()) % 16 == 0, what, ": out is not 16-byte aligned");
    at::assert_no_partial_overlap(*out_, query);
    at::assert_no_overlap(*out_, cache);
  }
  const OptionalHIPGuardMasqueradingAsCUDA guard(query.device());
  Tensor out = out_ ? *out_ : torch::empty({tokens, heads, d}, query.options());
  if (tokens == 0 || seqs == 0) return out;
  if (block_tables.size(1) == 0) {  // no sequence has a block: every row sees nothing
    NEED(!query_start, "block_tables has no columns");
    return out.zero_();
  }
  const Tensor q = heads_of(query), lens = ints(seq_lens);
  const Tensor tables = block_tables.stride(1) == 1 || block_tables.size(1) == 1 ? block_tables : block_tables.contiguous();
  const Tensor start = query_start ? ints(*query_start) : Tensor();
  const size_t bytes = serving_attend_kv4_workspace_bytes((int)tokens, (int)seqs, (int)heads, (int)kv, (int)d,
                                                          (int)max_query_len, (int)max_seq_len, (int)window);
  const Tensor workspace = bytes ? torch::empty({(int64_t)bytes}, cache.options()) : Tensor();
  raise_for(serving_attend_kv4(q.data_ptr(), q.stride(0), q.stride(1), cache.data_ptr(), tables.data_ptr<int32_t>(),
                               tables.stride(0), (int)tables.size(1), lens.data_ptr<int32_t>(),
                               query_start ? start.data_ptr<int32_t>() : nullptr, out.data_ptr(), (int)tokens, (int)seqs,
                               (int)heads, (int)kv, (int)d, cache.size(0), (int)block_size, (float)scale, (int)window,
                               (int)max_query_len, (int)max_seq_len, bf16, bytes ? workspace.data_ptr() : nullptr, bytes,
                               getCurrentHIPStreamMasqueradingAsCUDA().stream()),
            what);
  if (out_) written(out);
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& token_ids, int64_t top_n) {
  const char* what = "token_logprobs";
  const auto type = logits.scalar_type();
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16 || type == at::kFloat, what,
              ": expected scalar type Half, BFloat16 or Float but found ", type, " for logits");
  typed(token_ids, at::kLong, what, "token_ids");
  NEED(logits.dim() == 2 && logits.size(1) > 0, "logits must be [rows, vocabulary], got ", shape_of(logits));
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  NEED(token_ids.dim() == 1 && token_ids.size(0) == rows, "token_ids must be [rows], got ", shape_of(token_ids));
  NEED(top_n >= 0 && top_n <= 64 && top_n <= vocab, "top_n must be from 0 to 64 and no more than the vocabulary, got ", top_n);
  NEED(rows <= kMostInt && vocab <= 64 * 32760, "a vocabulary has at most 2096640 tokens, and there are too many rows or tokens here");
  on_gpu(logits, logits, what, "logits");
  on_gpu(token_ids, logits, what, "token_ids");
  no_gradient(logits, what, "logits");
  const OptionalHIPGuardMasqueradingAsCUDA guard(logits.device());
  const auto floats = logits.options().dtype(at::kFloat);
  Tensor logprob = torch::empty({rows}, floats), entropy = torch::empty({rows}, floats);
  Tensor ids = torch::empty({rows, top_n}, token_ids.options()), top = torch::empty({rows, top_n}, floats);
  if (rows == 0) return {logprob, entropy, ids, top};
  const Tensor x = logits.stride(1) == 1 || vocab == 1 ? logits : logits.contiguous(), given = ints(token_ids);
  const int kind = type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : 2;
  const size_t bytes = serving_token_logprobs_workspace_bytes((int)rows, (int)vocab, (int)top_n, kind);
  const Tensor workspace = bytes ? torch::empty({(int64_t)bytes}, logits.options().dtype(at::kByte)) : Tensor();
  raise_for(serving_token_logprobs(x.data_ptr(), x.stride(0), given.data_ptr<int64_t>(), logprob.data_ptr<float>(),
                                   entropy.data_ptr<float>(), top_n ? ids.data_ptr<int64_t>() : nullptr,
                                   top_n ? top.data_ptr<float>() : nullptr, (int)rows, (int)vocab, (int)top_n, kind,
                                   bytes ? workspace.data_ptr() : nullptr, bytes,
                                   getCurrentHIPStreamMasqueradingAsCUDA().stream()),
            what);
  return {logprob, entropy, ids, top};
}

}  // namespace

void bind_serving_ops(pybind11::module& ops) {
  namespace py = pybind11;
  ops.def("rope_append_kv4", &rope_append_kv4, py::arg("positions"), py::arg("query"), py::arg("key"), py::arg("value"),
          py::arg("cos_sin"), py::arg("cache"), py::arg("slots"), py::arg("interleaved") = false,
          "Rotates queries and keys, appends keys and values to a 4-bit paged cache");
  ops.def("kv4_read", &kv4_read, py::arg("cache"), py::arg("slots"), py::arg("head_size"), py::arg("dtype"),
          "Rows of a 4-bit paged cache as values");
  ops.def("paged_attention_kv4", &paged_attention_kv4, py::arg("query"), py::arg("cache"), py::arg("block_tables"),
          py::arg("seq_lens"), py::arg("scale"), py::arg("max_seq_len"), py::arg("query_start") = py::none(),
          py::arg("max_query_len") = 1, py::arg("window") = 0, py::arg("out") = py::none(),
          "Attention over a 4-bit paged cache");
  ops.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("token_ids"), py::arg("top_n") = 0,
          "Log probabilities of given tokens, entropy, most likely tokens");
}
