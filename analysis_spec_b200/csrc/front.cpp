// Torch front end of the decode-step operators (paged cache, token log-probabilities), as a
// CPython module: argument checks, outputs and workspaces from torch's allocator on the current
// stream, then one call of the C ABI. A decode step makes these calls once per layer and token,
// at sizes whose kernels run for a few microseconds, so the host side of a call is what it costs:
// a call through the same checks in Python and ctypes takes 22 to 32 us, here 5 to 8.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <array>

#include "../../include/speckv.h"

namespace py = pybind11;
using at::Tensor;
typedef std::optional<Tensor> Maybe;

namespace {

[[noreturn]] void value_error(const char* fn, const std::string& what) {
  throw py::value_error(std::string(fn) + ": " + what);
}

// Non-zero status of the C ABI as the package's SpecKVError.
void check_status(const char* name, int status) {
  if (status == SPECKV_OK) return;
  const std::string message = speckv_last_error();
  if (!PyGILState_Check())  // the autograd engine's thread
    throw std::runtime_error(std::string(name) + " failed (status " + std::to_string(status) + "): " + message);
  py::object type = py::module_::import("analysis_spec_b200._lib").attr("SpecKVError");
  py::object error = type(name, status, message);
  PyErr_SetObject(type.ptr(), error.ptr());
  throw py::error_already_set();
}

int dtype_code(const char* fn, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPECKV_F32;
    case at::kBFloat16: return SPECKV_BF16;
    case at::kHalf: return SPECKV_F16;
    default: value_error(fn, std::string("unsupported dtype ") + c10::toString(t));
  }
}

// Every tensor on the GPU of the first; returns its index.
int one_device(const char* fn, std::initializer_list<const Tensor*> tensors) {
  int dev = -1;
  for (const Tensor* t : tensors) {
    if (t == nullptr) continue;
    if (!t->is_cuda())
      throw std::runtime_error("analysis_spec_b200 kernels need CUDA tensors; got a tensor on " + t->device().str() +
                               " (the product has no CPU path)");
    if (dev < 0) dev = t->get_device();
    if (t->get_device() != dev)
      value_error(fn, "tensors on cuda:" + std::to_string(dev) + " and " + t->device().str());
  }
  return dev;
}

const Tensor* get(const Maybe& t) { return t.has_value() && t->defined() ? &*t : nullptr; }
const void* data(const Tensor* t) { return t != nullptr ? t->const_data_ptr() : nullptr; }
const int64_t* data64(const Tensor* t) { return static_cast<const int64_t*>(data(t)); }
// A new tensor on the GPU of `like`, without the dispatcher.
Tensor empty_like_device(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

void check_pages(const char* fn, const Tensor& k, const Tensor& v, const Tensor& table, int64_t batch) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
    value_error(fn, "key and value pages must be (pages, kv_heads, page_size, head_dim) of one dtype");
  if (k.stride(3) != 1 || v.stride(3) != 1) value_error(fn, "pages need unit stride on head_dim");
  if (table.scalar_type() != at::kLong || table.dim() != 2 || table.size(0) < batch ||
      (table.size(1) > 1 && table.stride(1) != 1))
    value_error(fn, "page table must be an int64 (batch, pages) tensor with unit column stride");
}

void per_sequence(const char* fn, const char* name, const Tensor& t, int64_t batch) {
  if (t.scalar_type() != at::kLong || t.dim() != 1 || t.size(0) < batch || (batch > 1 && t.stride(0) != 1))
    value_error(fn, std::string(name) + " must be a contiguous int64 tensor with an entry per sequence");
}

Maybe paged_append(const Tensor& key, const Tensor& value, const Tensor& key_pages, const Tensor& value_pages,
                   const Tensor& page_table, const Tensor& starts, const Maybe& counts_, const Maybe& query_,
                   const Maybe& cos_, const Maybe& sin_, const Maybe& positions_, bool interleaved,
                   const Maybe& query_out_) {
  const char* fn = "paged_append";
  const Tensor *counts = get(counts_), *query = get(query_), *cos = get(cos_), *sin = get(sin_),
               *positions = get(positions_), *out = get(query_out_);
  if (key.dim() != 4 || key.sizes() != value.sizes())
    value_error(fn, "key and value must be (batch, kv_heads, rows, head_dim) of one shape");
  const int64_t batch = key.size(0), kv_heads = key.size(1), rows = key.size(2), dim = key.size(3);
  check_pages(fn, key_pages, value_pages, page_table, batch);
  const at::ScalarType dtype = key_pages.scalar_type();
  const int code = dtype_code(fn, dtype);
  if (key.scalar_type() != dtype || value.scalar_type() != dtype)
    value_error(fn, "key / value dtype differs from the pages");
  if (key_pages.size(1) != kv_heads || key_pages.size(3) != dim)
    value_error(fn, "key / value shape does not match the pages");
  if (key.stride(3) != 1 || value.stride(3) != 1) value_error(fn, "key and value need unit stride on head_dim");
  per_sequence(fn, "starts", starts, batch);
  if (counts != nullptr) per_sequence(fn, "counts", *counts, batch);
  if (positions != nullptr && (positions->scalar_type() != at::kLong || positions->dim() != 2 ||
                               positions->size(0) < batch || positions->size(1) < rows))
    value_error(fn, "positions must be an int64 (batch, rows) tensor");
  int64_t rot = 0, rot_positions = 0;
  if (cos != nullptr || sin != nullptr) {
    if (cos == nullptr || sin == nullptr || cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat ||
        cos->dim() != 2 || cos->sizes() != sin->sizes() || !cos->is_contiguous() || !sin->is_contiguous())
      value_error(fn, "rotation must be a pair of contiguous float32 (positions, rotation_dim / 2) tables");
    rot_positions = cos->size(0);
    rot = 2 * cos->size(1);
    if (rot < 2 || rot > dim || rot_positions < 1)
      value_error(fn, "rotation of " + std::to_string(rot) + " of " + std::to_string(dim) + " dims over " +
                          std::to_string(rot_positions) + " positions");
  }
  if (query != nullptr) {
    if (query->dim() != 4 || query->size(0) != batch || query->size(2) != rows || query->size(3) != dim ||
        query->scalar_type() != dtype)
      value_error(fn, "query must be (batch, q_heads, rows, head_dim) of the pages' dtype");
    if (query->stride(3) != 1) value_error(fn, "query needs unit stride on head_dim");
    if (out != nullptr && (out->sizes() != query->sizes() || out->scalar_type() != dtype || out->stride(3) != 1))
      value_error(fn, "query and its output need one shape and dtype and unit stride on head_dim");
  } else if (out != nullptr) {
    value_error(fn, "query_out without query");
  }
  for (const Tensor* written : {&key_pages, &value_pages, out})  // expanded: rows would be stored over each other
    if (written != nullptr && at::has_internal_overlap(*written) == at::MemOverlap::Yes)
      value_error(fn, "the pages and query_out are written and must not overlap themselves (an expanded tensor does)");
  const int dev = one_device(fn, {&key, &value, &key_pages, &value_pages, &page_table, &starts, counts, query, cos, sin,
                                  positions, out});
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  Tensor made;
  if (query != nullptr && out == nullptr) {
    // (batch, rows, heads, dim) in memory, as projections and the attention lay their rows out
    made = empty_like_device({batch, rows, query->size(1), dim}, dtype, *query).transpose(1, 2);
    out = &made;
  }
  Maybe result;
  if (out != nullptr) result = *out;
  if (batch == 0 || rows == 0) return result;
  std::array<int64_t, 18> st{};
  for (int i = 0; i < 3; ++i) {
    st[i] = key.stride(i);
    st[3 + i] = value.stride(i);
    if (query != nullptr) {
      st[6 + i] = query->stride(i);
      st[9 + i] = out->stride(i);
    }
    st[12 + i] = key_pages.stride(i);
    st[15 + i] = value_pages.stride(i);
  }
  check_status("speckv_paged_append",
               speckv_paged_append(key.const_data_ptr(), value.const_data_ptr(), data(query),
                                   out != nullptr ? out->mutable_data_ptr() : nullptr, key_pages.mutable_data_ptr(),
                                   value_pages.mutable_data_ptr(), st.data(), data64(&page_table), page_table.stride(0),
                                   page_table.size(1), key_pages.size(0), key_pages.size(2), data64(&starts),
                                   data64(counts), data64(positions), positions != nullptr ? positions->stride(0) : 0,
                                   positions != nullptr ? positions->stride(1) : 0,
                                   static_cast<const float*>(data(cos)), static_cast<const float*>(data(sin)),
                                   rot_positions, rot, interleaved ? 1 : 0, batch,
                                   query != nullptr ? query->size(1) : 0, kv_heads, rows, dim, code, stream_of(dev)));
  return result;
}

Tensor paged_attention(const Tensor& query, const Tensor& key_pages, const Tensor& value_pages,
                       const Tensor& page_table, const Tensor& lengths, double scale, const Maybe& out_) {
  const char* fn = "paged_attention";
  const Tensor* given = get(out_);
  if (query.dim() != 4 || query.size(2) != 1)
    value_error(fn, "query must be (batch, q_heads, 1, head_dim): one new token per sequence");
  const int64_t batch = query.size(0), q_heads = query.size(1), dim = query.size(3);
  check_pages(fn, key_pages, value_pages, page_table, batch);
  const int code = dtype_code(fn, query.scalar_type());
  const int64_t kv_heads = key_pages.size(1);
  if (key_pages.scalar_type() != query.scalar_type() || key_pages.size(3) != dim || kv_heads < 1 ||
      q_heads % kv_heads != 0)
    value_error(fn, "query dtype, head_dim or heads do not match the pages");
  per_sequence(fn, "lengths", lengths, batch);
  if (query.stride(3) != 1) value_error(fn, "query needs unit stride on head_dim");
  if (given != nullptr &&
      (given->dim() != 4 || given->size(0) != batch || given->size(1) != 1 || given->size(2) != q_heads ||
       given->size(3) != dim || given->scalar_type() != query.scalar_type() || !given->is_contiguous()))
    value_error(fn, "out must be a contiguous (batch, 1, q_heads, head_dim) tensor of the query dtype");
  const int dev = one_device(fn, {&query, &key_pages, &value_pages, &page_table, &lengths, given});
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  Tensor out = given != nullptr ? *given : empty_like_device({batch, 1, q_heads, dim}, query.scalar_type(), query);
  if (batch == 0) return out;
  // a workspace of this call alone: other streams and captured graphs have their own
  const int64_t need = speckv_paged_attention_workspace(batch, q_heads, kv_heads, dim, page_table.size(1),
                                                        key_pages.size(2), code);
  Tensor workspace;
  if (need > 0) workspace = empty_like_device({need}, at::kByte, query);
  const int64_t st[8] = {query.stride(0),       query.stride(1),       key_pages.stride(0),   key_pages.stride(1),
                         key_pages.stride(2),   value_pages.stride(0), value_pages.stride(1), value_pages.stride(2)};
  check_status("speckv_paged_attention",
               speckv_paged_attention(query.const_data_ptr(), key_pages.const_data_ptr(), value_pages.const_data_ptr(),
                                      st, data64(&page_table), page_table.stride(0), page_table.size(1),
                                      key_pages.size(0), key_pages.size(2), data64(&lengths), out.mutable_data_ptr(),
                                      batch, q_heads, kv_heads, dim, (float)scale, code,
                                      need > 0 ? workspace.mutable_data_ptr() : nullptr, need, stream_of(dev)));
  return out;
}

// ---- token log-probabilities -------------------------------------------------------------------

struct Rows {
  int64_t batch = 1, per = 1, source = 1;
  int64_t logits[2] = {0, 0}, tokens[2] = {0, 0}, rows[2] = {0, 0};  // (sequence, row) strides
};

// Strides of a tensor whose leading dims are (), (rows,) or (batch, rows).
void lead_strides(const Tensor& t, int64_t lead, int64_t (&st)[2]) {
  if (lead == 1) st[1] = t.stride(0);
  if (lead == 2) {
    st[0] = t.stride(0);
    st[1] = t.stride(1);
  }
}

Rows check_rows(const char* fn, const Tensor& logits, const Tensor* tokens, const Tensor* rows, int64_t top,
                double temperature) {
  Rows r;
  dtype_code(fn, logits.scalar_type());
  const int64_t lead = logits.dim() - 1;
  if (lead < 0 || lead > 2 || logits.size(lead) < 1 || (logits.size(lead) > 1 && logits.stride(lead) != 1))
    value_error(fn, "logits must be ([batch,] [rows,] vocabulary) with unit stride on the vocabulary");
  const int64_t vocab = logits.size(lead);
  if (top < 0 || top > SPECKV_MAX_TOP || top > vocab)
    value_error(fn, std::to_string(top) + " alternatives of " + std::to_string(vocab) + " (at most " +
                        std::to_string(SPECKV_MAX_TOP) + ")");
  if (!(temperature >= 1e-29 && temperature <= 1e29))
    value_error(fn, "temperature must be positive and finite (1e-29 to 1e29), got " + std::to_string(temperature));
  if (lead == 1) r.source = logits.size(0);
  if (lead == 2) {
    r.batch = logits.size(0);
    r.source = logits.size(1);
  }
  r.per = r.source;
  at::IntArrayRef shape = logits.sizes().slice(0, lead);
  if (rows != nullptr) {
    if (lead != 2 || rows->dim() != 2 || rows->scalar_type() != at::kLong || rows->size(0) != r.batch)
      value_error(fn, "rows must be an int64 (batch, n) tensor beside (batch, rows, vocabulary) logits");
    shape = rows->sizes();
    r.per = rows->size(1);
    lead_strides(*rows, 2, r.rows);
  }
  if (tokens != nullptr) {
    if (tokens->scalar_type() != at::kLong || tokens->sizes() != shape)
      value_error(fn, "tokens must be int64 of the rows' shape");
    lead_strides(*tokens, lead, r.tokens);
  }
  lead_strides(logits, lead, r.logits);
  return r;
}

struct Scores {
  Tensor logprobs, entropy, stats, top_logprobs, top_ids;  // undefined: not asked for
};

Scores forward_scores(const Tensor& logits, const Tensor* tokens, const Tensor* rows, int64_t top, double temperature,
                      bool gradient) {
  const char* fn = "token_logprobs";
  const Rows r = check_rows(fn, logits, tokens, rows, top, temperature);
  const int dev = one_device(fn, {&logits, tokens, rows});
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  const at::IntArrayRef shape = rows != nullptr ? rows->sizes() : logits.sizes().slice(0, logits.dim() - 1);
  Scores s;
  c10::SmallVector<int64_t, 4> wide(shape.begin(), shape.end());
  if (tokens != nullptr) s.logprobs = empty_like_device(shape, at::kFloat, logits);
  s.entropy = empty_like_device(shape, at::kFloat, logits);
  wide.push_back(2);
  if (gradient) s.stats = empty_like_device(wide, at::kFloat, logits);
  if (top > 0) {
    wide.back() = top;
    s.top_logprobs = empty_like_device(wide, at::kFloat, logits);
    s.top_ids = empty_like_device(wide, at::kLong, logits);
  }
  check_status("speckv_token_logprobs",
               speckv_token_logprobs(logits.const_data_ptr(), dtype_code(fn, logits.scalar_type()), r.logits[0],
                                     r.logits[1], data64(tokens), r.tokens[0], r.tokens[1], data64(rows), r.rows[0],
                                     r.rows[1], r.batch, r.per, r.source, logits.size(-1), (float)(1.0 / temperature),
                                     (int32_t)top, tokens != nullptr ? s.logprobs.mutable_data_ptr<float>() : nullptr,
                                     s.entropy.mutable_data_ptr<float>(), gradient ? s.stats.mutable_data_ptr<float>() : nullptr,
                                     top > 0 ? s.top_logprobs.mutable_data_ptr<float>() : nullptr,
                                     top > 0 ? s.top_ids.mutable_data_ptr<int64_t>() : nullptr, stream_of(dev)));
  return s;
}

Tensor backward_scores(const Tensor& logits, const Tensor* tokens, const Tensor& entropy, const Tensor& stats,
                       const Tensor* top_ids, double temperature, Tensor g_logprobs, Tensor g_entropy, Tensor g_top) {
  const char* fn = "token_logprobs_backward";
  const int64_t top = top_ids != nullptr ? top_ids->size(-1) : 0;
  const Rows r = check_rows(fn, logits, tokens, nullptr, top, temperature);
  for (Tensor* g : {&g_logprobs, &g_entropy, &g_top})
    if (g->defined()) *g = g->to(at::kFloat).contiguous();  // expanded gradients of sums and means
  const Tensor* given[3];
  int i = 0;
  for (Tensor* g : {&g_logprobs, &g_entropy, &g_top}) given[i++] = g->defined() ? g : nullptr;
  const int dev = one_device(fn, {&logits, tokens, &entropy, &stats, top_ids, given[0], given[1], given[2]});
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  Tensor grad = empty_like_device(logits.sizes(), logits.scalar_type(), logits);
  check_status("speckv_token_logprobs_backward",
               speckv_token_logprobs_backward(
                   logits.const_data_ptr(), dtype_code(fn, logits.scalar_type()), r.logits[0], r.logits[1],
                   data64(tokens), r.tokens[0], r.tokens[1], r.batch, r.per, logits.size(-1),
                   (float)(1.0 / temperature), (int32_t)top, static_cast<const float*>(data(&entropy)),
                   static_cast<const float*>(data(&stats)), data64(top_ids), static_cast<const float*>(data(given[0])),
                   static_cast<const float*>(data(given[1])), static_cast<const float*>(data(given[2])),
                   grad.mutable_data_ptr(), stream_of(dev)));
  return grad;
}

// Outputs in the order logprobs (with tokens), entropy, then top_logprobs and top_ids (with top).
struct ScoreFunction : public torch::autograd::Function<ScoreFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits,
                                                const Maybe& tokens, int64_t top, double temperature) {
    Scores s = forward_scores(logits, get(tokens), nullptr, top, temperature, true);
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["tokens"] = get(tokens) != nullptr;
    ctx->set_materialize_grads(false);
    torch::autograd::variable_list out;
    if (s.logprobs.defined()) out.push_back(s.logprobs);
    out.push_back(s.entropy);
    if (top > 0) {
      out.push_back(s.top_logprobs);
      out.push_back(s.top_ids);
      ctx->mark_non_differentiable({s.top_ids});
    }
    ctx->save_for_backward({logits, get(tokens) != nullptr ? *tokens : Tensor(), s.entropy, s.stats, s.top_ids});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool tokens = ctx->saved_data["tokens"].toBool();
    const size_t at = tokens ? 1 : 0;
    const Tensor g_logprobs = tokens ? grads[0] : Tensor(), g_entropy = grads[at],
                 g_top = grads.size() > at + 1 ? grads[at + 1] : Tensor();
    Tensor grad;
    if (g_logprobs.defined() || g_entropy.defined() || g_top.defined()) {
      at::NoGradGuard no_grad;
      grad = backward_scores(saved[0].detach(), tokens ? &saved[1] : nullptr, saved[2].detach(), saved[3],
                             saved[4].defined() ? &saved[4] : nullptr, ctx->saved_data["temperature"].toDouble(),
                             g_logprobs, g_entropy, g_top);
    }
    if (grad.defined() && at::GradMode::is_enabled()) {  // create_graph: an error where it is differentiated again
      auto error = std::make_shared<torch::autograd::DelayedError>("token_logprobs is not twice differentiable", 2);
      torch::autograd::variable_list in{grad, saved[0]};  // on the way from the gradient to the logits
      grad = (*error)(std::move(in))[0];
    }
    return {grad, Tensor(), Tensor(), Tensor()};
  }
};

// A captured backward pass joins the stream on which a leaf's gradient is accumulated. Where a graph outside
// the capture keeps that node alive on another stream, the join breaks the capture from within the autograd
// engine and the process ends: refused while that can still be an error.
void check_capture(const Tensor& logits) {
  if (!logits.is_cuda() || !logits.is_leaf()) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(logits);
  if (node == nullptr) return;
  const auto stream = node->stream();
  if (stream.has_value() && *stream != c10::cuda::getCurrentCUDAStream(logits.get_device()).unwrap())
    throw std::runtime_error("token_logprobs: these logits are a leaf of an autograd graph made outside this capture, "
                             "which is still alive; drop its outputs first");
}

py::tuple token_logprobs(const Tensor& logits, const Maybe& tokens, const Maybe& rows, int64_t top,
                         double temperature) {
  auto item = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
  if (logits._fw_grad(0).defined())
    value_error("token_logprobs", "no forward-mode derivative: the logits carry a tangent, which would be lost");
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    if (get(rows) != nullptr)
      value_error("token_logprobs", "rows selects verified rows of a rollout and carries no gradient; detach the "
                                    "logits or index them first");
    check_capture(logits);
    const auto out = ScoreFunction::apply(logits, tokens, top, temperature);
    const size_t at = get(tokens) != nullptr ? 1 : 0;
    return py::make_tuple(at ? item(out[0]) : py::none(), item(out[at]), top > 0 ? item(out[at + 1]) : py::none(),
                          top > 0 ? item(out[at + 2]) : py::none());
  }
  const Scores s = forward_scores(logits, get(tokens), get(rows), top, temperature, false);
  return py::make_tuple(item(s.logprobs), item(s.entropy), item(s.top_logprobs), item(s.top_ids));
}

}  // namespace

PYBIND11_MODULE(_front, m) {
  m.def("paged_append", &paged_append);
  m.def("paged_attention", &paged_attention);
  m.def("token_logprobs", &token_logprobs);
}
