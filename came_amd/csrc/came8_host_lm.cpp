// The operators around the gated feed-forward block as autograd nodes: embedding, norm, 8-bit rows and their product, token log
// probabilities.  Natively, since host time is what a decoded token's small calls and a backward pass's many nodes cost.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/impl/VirtualGuardImpl.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <utility>
#include <vector>

#include "came8_host.h"

namespace came8_host {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------------------------------------------- operands
void not_traced(const char* op) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), op, ": cannot be traced; a trace would hold the result's allocation alone");
}

// The tensor behind an argument: strided, on the GPU, with its values in its own storage and no tangent
at::Tensor operand(const char* op, const char* name, PyObject* o) {
  TORCH_CHECK(THPVariable_Check(o), op, ": came_amd runs on the GPU; ", name, " is ", Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  const c10::DispatchKeySet keys = t.key_set();
  TORCH_CHECK(!keys.has(c10::DispatchKey::Python) && !keys.has(c10::DispatchKey::FuncTorchBatched) &&
                  !keys.has(c10::DispatchKey::FuncTorchGradWrapper) && !keys.has(c10::DispatchKey::Functionalize),
              op, ": ", name, " is a tensor subclass or of a function transform: its values may lie elsewhere");
  TORCH_CHECK(!t._fw_grad(0).defined(), op, ": no forward-mode derivatives; ", name, " has a tangent");
  TORCH_CHECK(t.is_cuda(), op, ": came_amd runs on the GPU; ", name, " is a ", t.device(), " tensor");
  TORCH_CHECK(t.layout() == at::kStrided, op, ": ", name, " is not strided");
  return t;
}
std::optional<at::Tensor> optional_operand(const char* op, const char* name, PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return operand(op, name, o);
}

void check_floating(const char* op, const char* name, const at::Tensor& t) {
  TORCH_CHECK(dtype_code(t) >= 0, op, ": unsupported dtype ", dtype_name(t), " of ", name,
              " (float32, bfloat16 and float16 are supported)");
}
void check_type(const char* op, const char* name, const at::Tensor& t, at::ScalarType type) {
  TORCH_CHECK(t.scalar_type() == type, op, ": ", name, " must be ", c10::toString(type), ", is ", dtype_name(t));
}
// of the type and device of `like`
void check_alike(const char* op, const char* name, const at::Tensor& t, const char* like_name, const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == like.scalar_type() && t.device() == like.device(), op, ": ", name, " is ", dtype_name(t), " on ",
              t.device(), ", ", like_name, " is ", dtype_name(like), " on ", like.device());
}
void check_device(const char* op, const char* name, const at::Tensor& t, const char* like_name, const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(), ", ", like_name, " on ", like.device());
}
void check_tokens(const char* op, const at::Tensor& t, const char* like_name, const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, op, ": tokens must be int64 or int32, are ", dtype_name(t));
  check_device(op, "tokens", t, like_name, like);
}
void no_gradient(const char* op, std::initializer_list<std::optional<at::Tensor>> operands) {
  if (!at::GradMode::is_enabled()) return;
  for (const auto& t : operands)
    TORCH_CHECK(!t || !t->requires_grad(), op, ": has no gradient; call it under torch.no_grad() or with detached operands");
}

bool has(const std::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }

// t [..., n] as rows [count, n] that are contiguous and do not overlap, at most `most` elements apart: itself where it lies so
struct Rows {
  at::Tensor t;
  int64_t count, ld;
};
Rows rows_of(const at::Tensor& t, int64_t most) {
  const int64_t n = t.size(-1), count = n > 0 ? t.numel() / n : 0;
  at::Tensor r = t.is_neg() ? t.resolve_neg() : t;
  if (r.dim() != 2) r = r.reshape({count, n});
  const bool fits = (n == 1 || r.stride(1) == 1) && (count <= 1 || (r.stride(0) >= n && r.stride(0) <= most));
  if (!fits) r = r.clone(at::MemoryFormat::Contiguous);
  return {r, count, count > 1 ? r.stride(0) : n};
}
constexpr int64_t kFar = int64_t(1) << 31;

at::Tensor plain(const at::Tensor& t) { return t.resolve_neg().contiguous(); }

// as many dimensions as t, the last of `width`
std::vector<int64_t> sizes_with(const at::Tensor& t, int64_t width) {
  std::vector<int64_t> s = t.sizes().vec();
  s.back() = width;
  return s;
}

c10::DataPtr workspace(size_t bytes) { return bytes > 0 ? c10::GetAllocator(at::kCUDA)->allocate(bytes) : c10::DataPtr(); }

void* stream_of(long long stream) { return reinterpret_cast<void*>(stream); }

// A parsed argument tuple
#define CAME8_PARSE(format, ...) \
  if (!PyArg_ParseTuple(args, format, __VA_ARGS__)) return nullptr

// ------------------------------------------------------------------------------------------------- embedding
came8_embedding embedding_of(const at::Tensor& tokens, const Rows& w, double scale, int64_t padding) {
  return came8_embedding{tokens.numel(), w.t.size(0), w.t.size(1), w.ld, padding, float(scale), dtype_code(w.t),
                         tokens.scalar_type() == at::kLong ? 8 : 4, 0};
}

at::Tensor embedding_forward(const at::Tensor& weight, const at::Tensor& tokens, double scale, int64_t padding, long long stream) {
  c10::OptionalDeviceGuard guard(weight.device());
  const at::Tensor t = plain(tokens);
  const Rows w = rows_of(weight, kFar);
  std::vector<int64_t> sizes = tokens.sizes().vec();
  sizes.push_back(weight.size(1));
  at::Tensor y = at::empty(sizes, weight.options());
  if (t.numel() > 0) {
    const came8_embedding e = embedding_of(t, w, scale, padding);
    entry_check(entries.embedding_forward(&e, t.data_ptr(), w.t.data_ptr(), y.data_ptr(), stream_of(stream)), "came8_embedding_forward");
  }
  return y;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& weight, const at::Tensor& tokens, double scale, int64_t padding,
                            int64_t stream, bool captured) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["sizes"] = weight.sizes();
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["stream"] = stream;  // the engine runs the backward pass on the forward's stream
    ctx->saved_data["captured"] = captured;
    return embedding_forward(weight, tokens, scale, padding, stream);
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    variable_list grads(6);
    if (!dys[0].defined()) return grads;
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    c10::OptionalDeviceGuard guard(dys[0].device());
    check_captured(ctx->saved_data["captured"].toBool(), "embedding", dys[0].device());
    const at::Tensor tokens = plain(ctx->get_saved_variables()[0]);
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const at::Tensor dy = plain(dys[0]);
    if (tokens.numel() == 0) {
      grads[0] = at::zeros(sizes, dy.options());
    } else {
      grads[0] = at::empty(sizes, dy.options());
      const came8_embedding e = embedding_of(tokens, Rows{grads[0], sizes[0], sizes[1]}, ctx->saved_data["scale"].toDouble(),
                                             ctx->saved_data["padding"].toInt());
      size_t bytes = 0;
      entry_check(entries.embedding_size(&e, &bytes), "came8_embedding_workspace_size");
      const c10::DataPtr ws = workspace(bytes);
      entry_check(entries.embedding_backward(&e, tokens.data_ptr(), dy.data_ptr(), grads[0].data_ptr(), ws.get(), bytes,
                                             stream_of(ctx->saved_data["stream"].toInt())),
                  "came8_embedding_backward");
    }
    if (again) grads[0] = differentiable_once({grads[0]}, "embedding")[0];
    return grads;
  }
};

// ------------------------------------------------------------------------------------------------------ norm
came8_rms_norm rms_of(const Rows& x, int64_t ld_residual, double eps) {
  return came8_rms_norm{x.count, x.t.size(1), x.ld, ld_residual, eps, dtype_code(x.t), 0};
}

// y, and h where there is a residual
variable_list rms_forward(const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& residual, double eps,
                          long long stream) {
  c10::OptionalDeviceGuard guard(x.device());
  const Rows r = rows_of(x, kFar);
  const at::Tensor w = plain(weight);
  at::Tensor y = at::empty(x.sizes(), x.options()), h;
  Rows res{};
  if (has(residual)) {
    res = rows_of(*residual, kFar);
    h = at::empty(x.sizes(), x.options());
  }
  if (r.count > 0) {
    const came8_rms_norm n = rms_of(r, res.ld, eps);
    entry_check(entries.rms_forward(&n, r.t.data_ptr(), res.t.defined() ? res.t.data_ptr() : nullptr, w.data_ptr(), y.data_ptr(),
                                    h.defined() ? h.data_ptr() : nullptr, stream_of(stream)),
                "came8_rms_norm_forward");
  }
  return h.defined() ? variable_list{y, h} : variable_list{y};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                               const std::optional<at::Tensor>& residual, double eps, int64_t stream, bool captured) {
    ctx->set_materialize_grads(false);
    variable_list out = rms_forward(x, weight, residual, eps, stream);
    ctx->save_for_backward({out.size() > 1 ? out[1] : x, weight});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["captured"] = captured;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const bool residual = dys.size() > 1;
    const at::Tensor dh = residual && dys[1].defined() ? dys[1] : at::Tensor();
    variable_list grads(6);
    if (!dys[0].defined() && !dh.defined()) return grads;
    const auto saved = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(saved[0].device());
    check_captured(ctx->saved_data["captured"].toBool(), "rms_norm", saved[0].device());
    const bool need_x = ctx->needs_input_grad(0) || (residual && ctx->needs_input_grad(2)), need_w = ctx->needs_input_grad(1);
    at::Tensor dx, dw;
    if (!dys[0].defined()) {  // h alone was used
      if (need_x) dx = dh;
    } else {
      const Rows h = rows_of(saved[0], kFar);
      if (need_w) dw = h.count > 0 ? at::empty(saved[1].sizes(), saved[1].options()) : at::zeros(saved[1].sizes(), saved[1].options());
      if (need_x) dx = at::empty(saved[0].sizes(), saved[0].options());
      if (h.count > 0) {
        const at::Tensor w = plain(saved[1]), dy = plain(dys[0]), dr = dh.defined() ? plain(dh) : dh;
        const came8_rms_norm n = rms_of(h, 0, ctx->saved_data["eps"].toDouble());
        size_t bytes = 0;
        c10::DataPtr ws;
        if (need_w) {
          entry_check(entries.rms_size(&n, &bytes), "came8_rms_norm_workspace_size");
          ws = workspace(bytes);
        }
        entry_check(entries.rms_backward(&n, h.t.data_ptr(), w.data_ptr(), dy.data_ptr(), dr.defined() ? dr.data_ptr() : nullptr,
                                         dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr, ws.get(), bytes,
                                         stream_of(ctx->saved_data["stream"].toInt())),
                    "came8_rms_norm_backward");
      }
    }
    if (again && (dx.defined() || dw.defined())) {
      const variable_list marked = differentiable_once({dx, dw}, "rms_norm");
      dx = marked[0];
      dw = marked[1];
    }
    if (ctx->needs_input_grad(0)) grads[0] = dx;
    grads[1] = dw;
    if (residual && ctx->needs_input_grad(2)) grads[2] = dx;
    return grads;
  }
};

void check_norm(const char* op, const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& residual, double eps) {
  check_floating(op, "x", x);
  check_alike(op, "weight", weight, "x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0 && weight.dim() == 1 && weight.size(0) == x.size(-1), op,
                    ": x [..., dim] and weight [dim]; got ", x.sizes(), " and ", weight.sizes());
  TORCH_CHECK_VALUE(std::isfinite(float(eps)) && eps >= 0.0, op, ": eps must be finite in float32 and at least 0, is ", eps);
  if (has(residual)) {
    check_alike(op, "residual", *residual, "x", x);
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), op, ": the residual has x's shape; got ", residual->sizes(), " and ", x.sizes());
  }
}

// codes [..., n] whose rows start at multiples of 16 bytes
at::Tensor empty_codes(const at::Tensor& x) {
  const int64_t n = x.size(-1);
  return at::empty(sizes_with(x, (n + 15) / 16 * 16), x.options().dtype(at::kChar)).narrow(-1, 0, n);
}
at::Tensor empty_scales(const at::Tensor& x) { return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)); }

// ------------------------------------------------------------------------------------------------ log probabilities
struct Tops {
  at::Tensor log_probs, tokens;
};

came8_log_probs log_probs_of(const Rows& z, const at::Tensor& tokens, int64_t top) {
  return came8_log_probs{z.count, z.t.size(1), z.ld, dtype_code(z.t), tokens.scalar_type() == at::kLong ? 8 : 4, int32_t(top), 0};
}

// log_probs, entropy and, with `keep`, what the backward pass takes beside them
variable_list log_probs_forward(const at::Tensor& logits, const at::Tensor& tokens, int64_t top, long long stream, bool keep, Tops* tops) {
  c10::OptionalDeviceGuard guard(logits.device());
  const Rows z = rows_of(logits, kFar);
  const at::Tensor t = plain(tokens);
  const at::TensorOptions f32 = logits.options().dtype(at::kFloat);
  const auto rows = tokens.sizes();
  at::Tensor lp = at::empty(rows, f32), entropy = at::empty(rows, f32), stats;
  if (keep) stats = at::empty({z.count, 2}, f32);
  std::vector<int64_t> sizes = rows.vec();
  sizes.push_back(top);
  tops->log_probs = at::empty(sizes, f32);
  tops->tokens = at::empty(sizes, logits.options().dtype(at::kLong));
  if (z.count > 0) {
    const came8_log_probs p = log_probs_of(z, t, top);
    size_t bytes = 0;
    entry_check(entries.logprob_size(&p, &bytes), "came8_log_probs_workspace_size");
    bytes = (bytes + 15) / 16 * 16;
    const c10::DataPtr ws = workspace(bytes + (keep ? 0 : size_t(z.count) * 8));
    float* m_and_l = keep ? stats.data_ptr<float>() : reinterpret_cast<float*>(static_cast<char*>(ws.get()) + bytes);
    entry_check(entries.logprob_forward(&p, z.t.data_ptr(), t.data_ptr(), lp.data_ptr<float>(), entropy.data_ptr<float>(), m_and_l,
                                        top > 0 ? tops->log_probs.data_ptr<float>() : nullptr,
                                        top > 0 ? tops->tokens.data_ptr<int64_t>() : nullptr, ws.get(), bytes, stream_of(stream)),
                "came8_log_probs_forward");
  }
  return {lp, entropy, stats};
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens, int64_t top, int64_t stream,
                               bool captured, Tops* tops) {
    ctx->set_materialize_grads(false);
    const variable_list out = log_probs_forward(logits, tokens, top, stream, true, tops);
    ctx->save_for_backward({logits, tokens, out[1], out[2]});
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["captured"] = captured;
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    variable_list grads(6);
    if (!dys[0].defined() && !dys[1].defined()) return grads;
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto saved = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(saved[0].device());
    check_captured(ctx->saved_data["captured"].toBool(), "token_log_probs", saved[0].device());
    const Rows z = rows_of(saved[0], kFar);
    const at::Tensor t = plain(saved[1]);
    grads[0] = at::empty(saved[0].sizes(), saved[0].options());
    if (z.count > 0) {
      const at::Tensor dlp = dys[0].defined() ? plain(dys[0]) : at::Tensor(), dent = dys[1].defined() ? plain(dys[1]) : at::Tensor();
      const came8_log_probs p = log_probs_of(z, t, 0);
      entry_check(entries.logprob_backward(&p, z.t.data_ptr(), t.data_ptr(), saved[3].data_ptr<float>(), saved[2].data_ptr<float>(),
                                           dlp.defined() ? dlp.data_ptr<float>() : nullptr, dent.defined() ? dent.data_ptr<float>() : nullptr,
                                           grads[0].data_ptr(), stream_of(ctx->saved_data["stream"].toInt())),
                  "came8_log_probs_backward");
    }
    if (again) grads[0] = differentiable_once({grads[0]}, "token_log_probs")[0];
    return grads;
  }
};

// the results as a tuple of Python's
PyObject* tuple_of(const variable_list& out) {
  PyObject* t = PyTuple_New(Py_ssize_t(out.size()));
  if (t == nullptr) return nullptr;
  for (size_t i = 0; i < out.size(); ++i) PyTuple_SET_ITEM(t, Py_ssize_t(i), THPVariable_Wrap(out[i]));
  return t;
}

}  // namespace

// -------------------------------------------------------------------------------------------- captured backwards
namespace {

// the leaf that an edge leads to, itself or (a reshaped, transposed or converted operand) through one node
template <typename F>
void each_leaf(const torch::autograd::Node& node, F&& f, bool through = true) {
  for (const auto& edge : node.next_edges()) {
    if (edge.function == nullptr) continue;
    if (auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) f(leaf);
    else if (through) each_leaf(*edge.function, f, false);
  }
}

// Whether a stream of the current device is being captured: a question of torch's about the current stream
bool captures(const c10::Stream& stream) {
  struct Current {
    c10::impl::VirtualGuardImpl impl;
    c10::Stream was;
    explicit Current(const c10::Stream& s) : impl(s.device_type()), was(impl.exchangeStream(s)) {}
    ~Current() { impl.exchangeStream(was); }
  } current(stream);
  pybind11::gil_scoped_acquire gil;
  return pybind11::module_::import("torch").attr("_C").attr("_cuda_isCurrentStreamCapturing")().cast<bool>();
}

}  // namespace

void check_captured(bool captured, const char* op, const at::Device& device) {
  if (!captured) return;
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  const auto* run = torch::autograd::get_current_graph_task_exec_info();
  const c10::Stream here = c10::impl::VirtualGuardImpl(device.type()).getStream(device);
  each_leaf(*node, [&](torch::autograd::AccumulateGrad* leaf) {
    if (run != nullptr && !run->empty()) {  // autograd.grad: no gradient is accumulated
      const auto found = run->find(leaf);
      if (found == run->end() || !found->second.needed_) return;
    }
    const auto its = leaf->stream();
    if (!its.has_value() || its->device() != here.device() || *its == here) return;
    TORCH_CHECK(captures(*its), op,
                ": a backward pass that is captured would accumulate a leaf's gradient on another stream: a graph of that leaf "
                "from outside of the capture is alive. Drop it before the capture, or run the warm-up on the capture's stream");
  });
}

// embedding(tokens, weight, scale: float, padding: int (-1: none), stream: int, captured: bool) -> y
PyObject* embedding(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *po_tokens, *po_weight;
  double scale;
  long long padding, stream;
  int captured;
  CAME8_PARSE("OOdLLp", &po_tokens, &po_weight, &scale, &padding, &stream, &captured);
  const char* op = "embedding";
  not_traced(op);
  const at::Tensor weight = operand(op, "weight", po_weight), tokens = operand(op, "tokens", po_tokens);
  check_floating(op, "weight", weight);
  check_tokens(op, tokens, "weight", weight);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.numel() > 0, op, ": weight [vocab, dim], not empty; got ", weight.sizes());
  TORCH_CHECK_VALUE(!std::isfinite(scale) || (std::isfinite(float(scale)) && (scale == 0.0 || float(scale) != 0.0f)), op,
                    ": float32 does not hold the scale ", scale);
  pybind11::gil_scoped_release no_gil;
  at::Tensor y = at::GradMode::is_enabled() && weight.requires_grad()
                     ? Embedding::apply(weight, tokens, scale, int64_t(padding), int64_t(stream), captured != 0)
                     : embedding_forward(weight, tokens, scale, padding, stream);
  pybind11::gil_scoped_acquire gil;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// rms_norm(x, weight, residual or None, eps: float, stream: int, captured: bool) -> (y,) or (y, h)
PyObject* rms_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *po_x, *po_w, *po_r;
  double eps;
  long long stream;
  int captured;
  CAME8_PARSE("OOOdLp", &po_x, &po_w, &po_r, &eps, &stream, &captured);
  const char* op = "rms_norm";
  not_traced(op);
  const at::Tensor x = operand(op, "x", po_x), w = operand(op, "weight", po_w);
  const std::optional<at::Tensor> r = optional_operand(op, "residual", po_r);
  check_norm(op, x, w, r, eps);
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (r && r->requires_grad())))
      out = RmsNorm::apply(x, w, r, eps, int64_t(stream), captured != 0);
    else
      out = rms_forward(x, w, r, eps, stream);
  }
  return tuple_of(out);
  END_HANDLE_TH_ERRORS
}

// rms_norm_int8(x, weight, residual or None, eps: float, stream: int) -> (q, scale) or (q, scale, h)
PyObject* rms_norm_int8(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *po_x, *po_w, *po_r;
  double eps;
  long long stream;
  CAME8_PARSE("OOOdL", &po_x, &po_w, &po_r, &eps, &stream);
  const char* op = "rms_norm_int8";
  not_traced(op);
  const at::Tensor x = operand(op, "x", po_x), w = operand(op, "weight", po_w);
  const std::optional<at::Tensor> r = optional_operand(op, "residual", po_r);
  check_norm(op, x, w, r, eps);
  no_gradient(op, {x, w, r});
  at::NoGradGuard no_grad;
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    c10::OptionalDeviceGuard guard(x.device());
    out = {empty_codes(x), empty_scales(x)};
    const Rows rows = rows_of(x, kFar);
    Rows res{};
    if (r) {
      res = rows_of(*r, kFar);
      out.push_back(at::empty(x.sizes(), x.options()));
    }
    if (rows.count > 0) {
      const at::Tensor weight = plain(w);
      const came8_rms_norm n = rms_of(rows, res.ld, eps);
      entry_check(entries.rms_int8(&n, rows.t.data_ptr(), r ? res.t.data_ptr() : nullptr, weight.data_ptr(), out[0].data_ptr<int8_t>(),
                                   (n.dim + 15) / 16 * 16, out[1].data_ptr<float>(), r ? out[2].data_ptr() : nullptr, stream_of(stream)),
                  "came8_rms_norm_int8");
    }
  }
  return tuple_of(out);
  END_HANDLE_TH_ERRORS
}

// quantize_rows(x, stream: int) -> (q, scale)
PyObject* quantize_rows(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* po_x;
  long long stream;
  CAME8_PARSE("OL", &po_x, &stream);
  const char* op = "quantize_rows";
  not_traced(op);
  const at::Tensor x = operand(op, "x", po_x);
  check_floating(op, "x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, op, ": x [..., dim]; got ", x.sizes());
  no_gradient(op, {x});
  at::NoGradGuard no_grad;
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    c10::OptionalDeviceGuard guard(x.device());
    out = {empty_codes(x), empty_scales(x)};
    const Rows rows = rows_of(x, kFar);
    if (rows.count > 0) {
      const came8_rms_norm n = rms_of(rows, 0, 0.0);
      entry_check(entries.quantize_rows(&n, rows.t.data_ptr(), out[0].data_ptr<int8_t>(), (n.dim + 15) / 16 * 16, out[1].data_ptr<float>(),
                                        stream_of(stream)),
                  "came8_quantize_rows");
    }
  }
  return tuple_of(out);
  END_HANDLE_TH_ERRORS
}

// int8_linear(q, scale, w_q, w_scale, bias or None, dtype: int, stream: int) -> y
PyObject* int8_linear(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *po_q, *po_s, *po_w, *po_ws, *po_b;
  int dtype;
  long long stream;
  CAME8_PARSE("OOOOOiL", &po_q, &po_s, &po_w, &po_ws, &po_b, &dtype, &stream);
  const char* op = "int8_linear";
  not_traced(op);
  const at::Tensor q = operand(op, "q", po_q), s = operand(op, "scale", po_s), w = operand(op, "w_q", po_w),
                   ws = operand(op, "w_scale", po_ws);
  const std::optional<at::Tensor> b = optional_operand(op, "bias", po_b);
  const at::ScalarType type = dtype == CAME8_F32 ? at::kFloat : dtype == CAME8_BF16 ? at::kBFloat16 : at::kHalf;
  check_type(op, "q", q, at::kChar);
  check_type(op, "w_q", w, at::kChar);
  check_type(op, "scale", s, at::kFloat);
  check_type(op, "w_scale", ws, at::kFloat);
  check_device(op, "scale", s, "q", q);
  check_device(op, "w_q", w, "q", q);
  check_device(op, "w_scale", ws, "q", q);
  TORCH_CHECK_VALUE(q.dim() >= 1 && w.dim() == 2 && q.size(-1) == w.size(1) && w.numel() > 0, op,
                    ": q [..., in] and w_q [out, in], not empty; got ", q.sizes(), " and ", w.sizes());
  TORCH_CHECK_VALUE(w.size(1) <= 131071, op, ": at most 131071 codes a row, whose sum fits 32 bits; got ", w.size(1));
  TORCH_CHECK_VALUE(s.sizes() == q.sizes().slice(0, q.dim() - 1) && ws.dim() == 1 && ws.size(0) == w.size(0), op,
                    ": a scale for each row of q and of w_q; got ", s.sizes(), " and ", ws.sizes());
  if (b) {
    check_type(op, "bias", *b, type);
    check_device(op, "bias", *b, "q", q);
    TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == w.size(0), op, ": bias [out]; got ", b->sizes());
  }
  no_gradient(op, {s, ws, b});
  at::NoGradGuard no_grad;
  at::Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    c10::OptionalDeviceGuard guard(q.device());
    y = at::empty(sizes_with(q, w.size(0)), q.options().dtype(type));
    auto codes_of = [](const at::Tensor& t) {  // rows that could all start on words do
      Rows r = rows_of(t, int64_t(1) << 20);
      if (r.ld % 4 == 0 && reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 4 != 0) {
        r.t = r.t.clone(at::MemoryFormat::Contiguous);
        r.ld = r.t.size(1);
      }
      return r;
    };
    const Rows rq = codes_of(q), rw = codes_of(w);
    if (rq.count > 0) {
      const at::Tensor scale = plain(s), w_scale = plain(ws), bias = b ? plain(*b) : at::Tensor();
      const came8_int8_linear l{rq.count, w.size(1), w.size(0), rq.ld, rw.ld, dtype, 0};
      size_t bytes = 0;
      entry_check(entries.int8_size(&l, &bytes), "came8_int8_linear_workspace_size");
      const c10::DataPtr space = workspace(bytes);
      entry_check(entries.int8_forward(&l, rq.t.data_ptr<int8_t>(), scale.data_ptr<float>(), rw.t.data_ptr<int8_t>(),
                                       w_scale.data_ptr<float>(), b ? bias.data_ptr() : nullptr, y.data_ptr(), space.get(), bytes,
                                       stream_of(stream)),
                  "came8_int8_linear_forward");
    }
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// token_log_probs(logits, tokens, top: int, stream: int, captured: bool) -> (log_probs, entropy, top_log_probs, top_tokens)
PyObject* token_log_probs(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *po_z, *po_t;
  long long top, stream;
  int captured;
  CAME8_PARSE("OOLLp", &po_z, &po_t, &top, &stream, &captured);
  const char* op = "token_log_probs";
  not_traced(op);
  const at::Tensor z = operand(op, "logits", po_z), tokens = operand(op, "tokens", po_t);
  check_floating(op, "logits", z);
  check_tokens(op, tokens, "logits", z);
  TORCH_CHECK_VALUE(z.dim() >= 1 && z.size(-1) > 0 && tokens.sizes() == z.sizes().slice(0, z.dim() - 1), op,
                    ": logits [..., vocab] and tokens [...]; got ", z.sizes(), " and ", tokens.sizes());
  TORCH_CHECK_VALUE(z.size(-1) <= (int64_t(1) << 20), op, ": a vocabulary of at most 2^20; got ", z.size(-1));
  TORCH_CHECK_VALUE(top >= 0 && top <= 64 && top <= z.size(-1), op, ": top must be in [0, 64] and at most the vocabulary; got ", top);
  Tops tops;
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled() && z.requires_grad())
      out = TokenLogProbs::apply(z, tokens, int64_t(top), int64_t(stream), captured != 0, &tops);
    else
      out = log_probs_forward(z, tokens, top, stream, false, &tops);
  }
  return tuple_of({out[0], out[1], tops.log_probs, tops.tokens});
  END_HANDLE_TH_ERRORS
}

}  // namespace came8_host
