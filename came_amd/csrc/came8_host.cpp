// came8_host: descriptors of a param group's tensors for came8_step, filled natively; AdamW's step and the gradient norm with
// theirs; and the gated feed-forward block as an autograd node.
//
// gather() does what the optimizers' Python does for every parameter of a group before a step (the checks of
// _prepare_param and _check_state, the fields of _descriptors and _fill_desc, the step counts) for the plain case:
// contiguous strided parameters and gradients on one GPU whose states exist in the optimizer's own layout.  It checks
// all of them anew on every call, changes nothing unless all pass, and returns None otherwise, upon which the Python
// takes the group from the start: it creates states, copies what is not contiguous and raises the errors.
// 192 adapters of 10 to 130 KB: 64 us of host time a step instead of 940; 292 tensors of a 24-layer model: 196 us
// instead of 1380.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>

#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include "../../include/came8.h"

namespace {

PyObject* key(const char* name) { return PyUnicode_InternFromString(name); }

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CAME8_F32;
    case at::kBFloat16: return CAME8_BF16;
    case at::kHalf: return CAME8_F16;
    default: return -1;
  }
}

// the tensor under `name` in a state, or null (borrowed)
const at::Tensor* tensor_of(PyObject* st, PyObject* name) {
  PyObject* o = PyDict_GetItemWithError(st, name);
  return o != nullptr && THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// A parameter's state (borrowed), or null.  A tensor's hash is its address (torch.Tensor.__hash__, which the lookup would
// call in Python for every parameter: CAME's gather of 192 tensors took 44 us so, and takes 30 without the calls).
PyObject* state_of(PyObject* state, PyObject* param) {
  return _PyDict_GetItem_KnownHash(state, param, Py_hash_t(reinterpret_cast<uintptr_t>(param)));
}

bool flag_off(PyObject* st, PyObject* name) {
  PyObject* o = PyDict_GetItemWithError(st, name);
  return o == nullptr || o == Py_False;
}

int64_t num_blocks(int64_t n, int64_t block) { return n <= 0 ? 1 : (n + block - 1) / block; }

template <typename T>
void put(T*& field, const at::Tensor* t) {
  field = static_cast<T*>(t->data_ptr());
}

// What the plain case asks of the parameter and gradient themselves.  The whole group is looked over before the first
// state is: a group that the Python takes after all (a transposed gradient at the end of 290 tensors) has then lost 8 us of
// its 1200, not 52.
bool plain(const at::Tensor& p, const at::Tensor& g) {
  return p.is_cuda() && p.layout() == at::kStrided && g.layout() == at::kStrided && g.device() == p.device() &&
         p.is_contiguous() && g.is_contiguous() && p.numel() != 0 && p.sizes() == g.sizes() && dtype_code(p) >= 0 &&
         dtype_code(g) >= 0;
}

// One parameter's descriptor; false: not the plain case.  *step: its state's step count.
bool describe(const at::Tensor& p, const at::Tensor& g, PyObject* st, int kind, int64_t block, came8_tensor& d,
              long* step) {
  static PyObject *k_mode = key("_mode"), *k_nd = key("_cuda_factored_nd_ext_path"),
                  *k_ndc = key("_cuda_factored_nd_chunked_ext_path"), *k_fact = key("factored"), *k_step = key("step"),
                  *k_mq = key("exp_avg_q"), *k_ma = key("exp_avg_absmax"), *k_rq = key("factored_row_q"),
                  *k_ra = key("factored_row_absmax"), *k_cq = key("factored_col_q"),
                  *k_ca = key("factored_col_absmax"), *k_vq = key("exp_avg_sq_q"), *k_va = key("exp_avg_sq_absmax"),
                  *k_m = key("exp_avg"), *k_v = key("exp_avg_sq"), *k_sr = key("exp_avg_sq_row"),
                  *k_sc = key("exp_avg_sq_col"), *k_rr = key("exp_avg_res_row"), *k_rc = key("exp_avg_res_col");
  PyObject* mode = PyDict_GetItemWithError(st, k_mode);
  if (mode == nullptr || !PyUnicode_Check(mode) ||
      PyUnicode_CompareWithASCIIString(mode, kind == CAME8_STATE_FP32 ? "cudafp" : "full8bit") != 0)
    return false;
  PyObject* fo = PyDict_GetItemWithError(st, k_fact);
  if (fo != Py_True && fo != Py_False) return false;
  const bool fact = fo == Py_True;
  const int64_t nd = p.dim(), n = p.numel();
  if (fact != (nd >= 2)) return false;
  PyObject* so = PyDict_GetItemWithError(st, k_step);
  if (so == nullptr || !PyLong_CheckExact(so)) return false;
  int over = 0;
  *step = PyLong_AsLongAndOverflow(so, &over);
  if (over != 0) return false;
  const int64_t C = nd > 0 ? p.size(nd - 1) : 1, R = fact ? p.size(nd - 2) : 1, P = fact ? n / (R * C) : 1;
  d = came8_tensor{};
  d.param = p.data_ptr();
  d.grad = g.data_ptr();
  d.param_dtype = dtype_code(p);
  d.grad_dtype = dtype_code(g);
  d.state_kind = kind;
  d.factored = fact ? 1 : 0;
  d.prefix = P;
  d.rows = R;
  d.cols = fact ? C : n;
  if (kind == CAME8_STATE_FP32) {
    const at::Tensor* m = tensor_of(st, k_m);
    if (m == nullptr || m->sizes() != p.sizes()) return false;
    const at::Tensor* s[5] = {m, fact ? tensor_of(st, k_sr) : tensor_of(st, k_v), fact ? tensor_of(st, k_rr) : m,
                              fact ? tensor_of(st, k_sc) : m, fact ? tensor_of(st, k_rc) : m};
    for (const at::Tensor* t : s)
      if (t == nullptr || t->device() != p.device() || t->scalar_type() != at::kFloat || !t->is_contiguous()) return false;
    put(d.exp_avg_q, s[0]);
    put(d.row_q, s[1]);
    if (fact) {
      put(d.row_absmax, s[2]);
      put(d.col_q, s[3]);
      put(d.col_absmax, s[4]);
    }
    return true;
  }
  if (!flag_off(st, k_nd) || !flag_off(st, k_ndc)) return false;  // per-matrix blocks
  const at::Tensor *mq = tensor_of(st, k_mq), *ma = tensor_of(st, k_ma);
  if (mq == nullptr || ma == nullptr || mq->sizes() != p.sizes() || mq->device() != p.device() ||
      ma->numel() != num_blocks(n, block))
    return false;
  put(d.exp_avg_q, mq);
  put(d.exp_avg_absmax, ma);
  const at::Tensor *rq = tensor_of(st, fact ? k_rq : k_vq), *ra = tensor_of(st, fact ? k_ra : k_va);
  if (rq == nullptr || ra == nullptr) return false;
  put(d.row_q, rq);
  put(d.row_absmax, ra);
  if (fact) {
    const at::Tensor *cq = tensor_of(st, k_cq), *ca = tensor_of(st, k_ca);
    if (cq == nullptr || ca == nullptr || rq->numel() != 2 * P * R || ra->numel() != 2 * num_blocks(P * R, block) ||
        cq->numel() != 2 * P * C || ca->numel() != 2 * num_blocks(P * C, block))
      return false;
    put(d.col_q, cq);
    put(d.col_absmax, ca);
  }
  return true;
}

// The parameters of a list that have a gradient, and the gradients; false: not the plain case.  The references to the
// gradients are kept: a key's hash may run Python, which may replace one.
bool collect(PyObject* params, int64_t cap, std::vector<PyObject*>& used, std::vector<at::Tensor>& grads) {
  const Py_ssize_t n = PyList_GET_SIZE(params);
  used.reserve(size_t(n));
  grads.reserve(size_t(n));
  const at::Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* po = PyList_GET_ITEM(params, i);
    if (!THPVariable_CheckExact(po)) return false;  // subclasses may keep their data elsewhere
    const at::Tensor& p = THPVariable_Unpack(po);
    const at::Tensor& g = p.grad();
    if (!g.defined()) continue;
    if (first == nullptr) first = &p;
    if (g.key_set().has(c10::DispatchKey::Python) || int64_t(used.size()) >= cap || p.device() != first->device() ||
        !plain(p, g))
      return false;
    used.push_back(po);
    grads.push_back(g);
  }
  return true;
}

// The list of `used`, every state's step count advanced by one; null with a Python error set.
PyObject* advanced(const std::vector<PyObject*>& used, const std::vector<std::pair<PyObject*, long>>& counts) {
  static PyObject* k_step = key("step");
  PyObject* res = PyList_New(Py_ssize_t(used.size()));
  if (res == nullptr) return nullptr;
  for (size_t i = 0; i < used.size(); ++i) {
    Py_INCREF(used[i]);
    PyList_SET_ITEM(res, Py_ssize_t(i), used[i]);
    PyObject* v = PyLong_FromLong(counts[i].second + 1);
    if (v == nullptr || PyDict_SetItem(counts[i].first, k_step, v) != 0) {
      Py_XDECREF(v);
      Py_DECREF(res);
      return nullptr;
    }
    Py_DECREF(v);
  }
  return res;
}

// gather(params: list, state: dict, address: int, capacity: int, state_kind: int, block_size: int)
//   -> list of the parameters with a gradient, whose came8_tensor descriptors now lie at `address` in that order and
//      whose step counts are advanced; None: not the plain case, nothing changed.
PyObject* gather(PyObject*, PyObject* args) {
  PyObject *params, *state;
  unsigned long long addr;
  long long cap, block;
  int kind;
  if (!PyArg_ParseTuple(args, "O!O!KLiL", &PyList_Type, &params, &PyDict_Type, &state, &addr, &cap, &kind, &block))
    return nullptr;
  if (block < 1) Py_RETURN_NONE;  // the blocks are counted by a division; the Python raises the error
  try {
    came8_tensor* out = reinterpret_cast<came8_tensor*>(static_cast<uintptr_t>(addr));
    std::vector<PyObject*> used;                     // the parameters with a gradient
    std::vector<std::pair<PyObject*, long>> counts;  // their states and step counts (the dicts outlive this call)
    std::vector<at::Tensor> grads;
    if (!collect(params, cap, used, grads)) Py_RETURN_NONE;
    counts.reserve(used.size());
    for (size_t i = 0; i < used.size(); ++i) {
      const at::Tensor& p = THPVariable_Unpack(used[i]);
      PyObject* st = state_of(state, used[i]);
      long step = 0;
      if (st == nullptr || !PyDict_Check(st) || !describe(p, grads[i], st, kind, block, out[i], &step)) {
        PyErr_Clear();
        Py_RETURN_NONE;
      }
      counts.emplace_back(st, step);
    }
    return advanced(used, counts);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// libcame8's entries, which Python has loaded
struct Entries {
  decltype(&came8_last_error) error = nullptr;
  decltype(&came8_adamw_step) adamw = nullptr;
  decltype(&came8_grad_norm_workspace_size) norm_size = nullptr;
  decltype(&came8_grad_norm) norm = nullptr;
  decltype(&came8_grad_clip) clip = nullptr;
  decltype(&came8_gated_ffn_workspace_size) ffn_size = nullptr;
  decltype(&came8_gated_ffn_forward) ffn_forward = nullptr;
  decltype(&came8_gated_ffn_backward) ffn_backward = nullptr;
} entries;

void entry_check(int rc, const char* what) { TORCH_CHECK(rc == CAME8_OK, what, " failed (", rc, "): ", entries.error()); }

// A tensor that a kernel has written, for the nodes that have saved it (gated_ffn its weights); inference tensors have no
// version.
void written(c10::TensorImpl* t) {
  if (!t->is_inference()) t->bump_version();
}

// The buffer of a moment or its scales: contiguous, of the parameter's device; null otherwise.
void* moment(PyObject* st, PyObject* name, const at::Tensor& p, at::ScalarType type, int64_t n) {
  const at::Tensor* t = tensor_of(st, name);
  return t != nullptr && t->scalar_type() == type && t->numel() == n && t->device() == p.device() && t->is_contiguous()
             ? t->data_ptr()
             : nullptr;
}

// adamw_step(params: list, state: dict, bits, block_size, seed, lr, beta1, beta2, eps, weight_decay, grad_scale: int, stream:
//   int) -> True: the group's parameters with a gradient are stepped (came8_adamw_step) and their step counts advanced;
//   None: not the plain case, nothing changed.  As gather(), and the call with it: 4 tensors 17 us of host time a step
//   instead of 19 with the descriptors handed back.
PyObject* adamw_step(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *params, *state;
  unsigned long long scale, stream;
  came8_adamw_hparams hp{};
  if (!PyArg_ParseTuple(args, "O!O!iiIdddddKK", &PyList_Type, &params, &PyDict_Type, &state, &hp.bits, &hp.block_size, &hp.seed,
                        &hp.lr, &hp.beta1, &hp.beta2, &hp.eps, &hp.weight_decay, &scale, &stream))
    return nullptr;
  if (hp.block_size < 1) Py_RETURN_NONE;
  static PyObject *k_step = key("step"), *k_m = key("exp_avg"), *k_v = key("exp_avg_sq"), *k_mq = key("exp_avg_q"),
                  *k_vq = key("exp_avg_sq_q"), *k_ma = key("exp_avg_absmax"), *k_va = key("exp_avg_sq_absmax");
  std::vector<PyObject*> used;
  std::vector<at::Tensor> grads;
  if (!collect(params, PyList_GET_SIZE(params), used, grads)) Py_RETURN_NONE;
  if (used.empty()) Py_RETURN_TRUE;
  std::vector<came8_adamw_tensor> descs(used.size());
  std::vector<std::pair<PyObject*, long>> counts;
  counts.reserve(used.size());
  for (size_t i = 0; i < used.size(); ++i) {
    const at::Tensor& p = THPVariable_Unpack(used[i]);
    PyObject* st = state_of(state, used[i]);
    PyObject* so = st != nullptr && PyDict_Check(st) ? PyDict_GetItemWithError(st, k_step) : nullptr;
    int over = 0;
    const long step = so != nullptr && PyLong_CheckExact(so) ? PyLong_AsLongAndOverflow(so, &over) : -1;
    if (step < 0 || over != 0 || grads[i].is_neg()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    came8_adamw_tensor& d = descs[i];
    d.param = p.data_ptr();
    d.grad = grads[i].data_ptr();
    d.numel = p.numel();
    d.step = step + 1;
    d.param_dtype = dtype_code(p);
    d.grad_dtype = dtype_code(grads[i]);
    if (hp.bits == 32) {
      d.exp_avg = moment(st, k_m, p, at::kFloat, d.numel);
      d.exp_avg_sq = moment(st, k_v, p, at::kFloat, d.numel);
    } else {
      d.exp_avg = moment(st, k_mq, p, at::kChar, d.numel);
      d.exp_avg_sq = moment(st, k_vq, p, at::kByte, d.numel);
      d.exp_avg_absmax = static_cast<float*>(moment(st, k_ma, p, at::kFloat, num_blocks(d.numel, hp.block_size)));
      d.exp_avg_sq_absmax = static_cast<float*>(moment(st, k_va, p, at::kFloat, num_blocks(d.numel, hp.block_size)));
    }
    if (d.exp_avg == nullptr || d.exp_avg_sq == nullptr ||
        (hp.bits != 32 && (d.exp_avg_absmax == nullptr || d.exp_avg_sq_absmax == nullptr))) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    counts.emplace_back(st, step);
  }
  c10::OptionalDeviceGuard guard(grads[0].device());
  entry_check(entries.adamw(descs.data(), int32_t(descs.size()), &hp, reinterpret_cast<const float*>(scale),
                            reinterpret_cast<void*>(stream)),
              "came8_adamw_step");
  for (PyObject* po : used) written(THPVariable_Unpack(po).unsafeGetTensorImpl());
  PyObject* list = advanced(used, counts);
  if (list == nullptr) return nullptr;
  Py_DECREF(list);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// grad_norm(tensors: list, of_parameters: bool, max_norm: float, scale: bool, stream: int) -> (norm, factor), device scalars of
//   the tensors (or of the parameters' gradients, of those that have one); with scale they are multiplied in place, and the
//   factor is None.  False: no tensors; None: some tensor is not a plain contiguous one of the first's device.
PyObject* grad_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* tensors;
  int of_parameters, scale;
  double max_norm;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "O!pdpK", &PyList_Type, &tensors, &of_parameters, &max_norm, &scale, &stream)) return nullptr;
  std::vector<came8_grad_tensor> descs;
  std::vector<c10::TensorImpl*> scaled;
  descs.reserve(size_t(PyList_GET_SIZE(tensors)));
  scaled.reserve(size_t(PyList_GET_SIZE(tensors)));
  at::Tensor first;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(tensors); ++i) {
    PyObject* o = PyList_GET_ITEM(tensors, i);
    if (!THPVariable_Check(o)) Py_RETURN_NONE;
    const at::Tensor& t = of_parameters ? THPVariable_Unpack(o).grad() : THPVariable_Unpack(o);
    if (of_parameters && !t.defined()) continue;
    if (!first.defined()) first = t;
    if (t.key_set().has(c10::DispatchKey::Python) || !t.is_cuda() || t.device() != first.device() || t.layout() != at::kStrided ||
        !t.is_contiguous() || dtype_code(t) < 0)
      Py_RETURN_NONE;
    descs.push_back(came8_grad_tensor{t.numel() > 0 ? t.data_ptr() : nullptr, t.numel(), dtype_code(t), 0});
    if (scale) scaled.push_back(t.unsafeGetTensorImpl());
  }
  if (descs.empty()) Py_RETURN_FALSE;
  c10::OptionalDeviceGuard guard(first.device());
  const int32_t n = int32_t(descs.size());
  const size_t bytes = entries.norm_size(n);
  const at::TensorOptions options = first.options().dtype(at::kFloat).requires_grad(false);
  // A program may keep every step's norm, which keeps no workspace.  That and a clip's factor are no tensors: the clip of 192
  // adapters takes 23.1 us so, 25.5 with both scalars views of one.
  const at::Tensor norm = at::empty({}, options);
  const at::Tensor factor = scale ? at::Tensor() : at::empty({}, options);
  const c10::DataPtr ws = c10::GetAllocator(at::kCUDA)->allocate(bytes + sizeof(float));
  float* own_factor = reinterpret_cast<float*>(static_cast<char*>(ws.get()) + bytes);
  entry_check((scale ? entries.clip : entries.norm)(descs.data(), n, max_norm, norm.data_ptr<float>(),
                                                    scale ? own_factor : factor.data_ptr<float>(), ws.get(), bytes,
                                                    reinterpret_cast<void*>(stream)),
              scale ? "came8_grad_clip" : "came8_grad_norm");
  for (c10::TensorImpl* t : scaled) written(t);
  if (scale) return Py_BuildValue("NO", THPVariable_Wrap(norm), Py_None);
  return Py_BuildValue("NN", THPVariable_Wrap(norm), THPVariable_Wrap(factor));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------- gated feed-forward block
// The block as an autograd node.  In Python its backward pass, which runs on a thread of the engine's, waits for the
// interpreter's lock twice: 198 us of host time for 4 tokens of 256 and 512 forward and backward, 81 natively.
std::string dtype_name(const at::Tensor& t) {
  const char* known[3] = {"torch.float32", "torch.bfloat16", "torch.float16"};
  const int code = dtype_code(t);
  return code >= 0 ? known[code] : c10::toString(t.scalar_type());
}

// A 2-D tensor whose rows are contiguous and do not overlap, at a 4-byte aligned address: itself, or a copy where it is not
// or where its rows lie too far apart for the kernels.
at::Tensor rows_of(const at::Tensor& t) {
  const int64_t n = t.size(1);
  const bool fits = (t.stride(1) == 1 || n == 1) && (t.size(0) == 1 || (t.stride(0) >= n && t.stride(0) <= (1 << 20))) &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 4 == 0 && !t.is_neg();
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct FfnOperands {
  at::Tensor x, gate, up, down;
  came8_ffn f;
};

FfnOperands ffn_operands(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const at::Tensor& down, int64_t act) {
  FfnOperands o{rows_of(x), rows_of(gate), rows_of(up), rows_of(down), {}};
  auto ld = [](const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); };
  o.f = came8_ffn{x.size(0), x.size(1), gate.size(0), down.size(0), ld(o.x), ld(o.gate), ld(o.up), ld(o.down), dtype_code(x),
                  int32_t(act)};
  return o;
}

at::Tensor ffn_workspace(const came8_ffn& f, bool backward, const at::Tensor& like, size_t* bytes) {
  entry_check(entries.ffn_size(&f, backward ? 1 : 0, bytes), "came8_gated_ffn_workspace_size");
  return at::empty({int64_t(*bytes)}, like.options().dtype(at::kByte));
}

// y, and g and u [2, tokens, hidden] where they are kept
std::pair<at::Tensor, at::Tensor> ffn_forward(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up,
                                              const at::Tensor& down, int64_t act, int64_t stream, bool keep) {
  c10::OptionalDeviceGuard guard(x.device());
  const FfnOperands o = ffn_operands(x, gate, up, down, act);
  const int64_t T = o.f.tokens, F = o.f.hidden;
  at::Tensor y = at::empty({T, o.f.out}, x.options()), gu;
  if (keep) gu = at::empty({2, T, F}, x.options().dtype(at::kFloat));
  if (T > 0) {
    size_t bytes = 0;
    const at::Tensor ws = ffn_workspace(o.f, false, x, &bytes);
    float* g = keep ? gu.data_ptr<float>() : nullptr;
    entry_check(entries.ffn_forward(&o.f, o.x.data_ptr(), o.gate.data_ptr(), o.up.data_ptr(), o.down.data_ptr(), y.data_ptr(), g,
                          keep ? g + T * F : nullptr, ws.data_ptr(), bytes, reinterpret_cast<void*>(stream)),
              "came8_gated_ffn_forward");
  }
  return {y, gu};
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up,
                            const at::Tensor& down, int64_t act, int64_t stream) {
    auto [y, gu] = ffn_forward(x, gate, up, down, act, stream, true);
    ctx->save_for_backward({x, gate, up, down, gu});
    ctx->saved_data["act"] = act;
    ctx->saved_data["stream"] = stream;  // the engine runs the backward pass on the forward's stream
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dys) {
    const bool again = at::GradMode::is_enabled();  // of gradients of gradients there are none
    at::NoGradGuard no_grad;
    const auto saved = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(saved[0].device());
    const FfnOperands o = ffn_operands(saved[0], saved[1], saved[2], saved[3], ctx->saved_data["act"].toInt());
    const int64_t T = o.f.tokens, F = o.f.hidden;
    const at::Tensor* ops[4] = {&saved[0], &saved[1], &saved[2], &saved[3]};
    torch::autograd::variable_list grads(6);
    for (size_t i = 0; i < 4; ++i)
      if (ctx->needs_input_grad(i))
        grads[i] = T > 0 ? at::empty(ops[i]->sizes(), ops[i]->options()) : at::zeros(ops[i]->sizes(), ops[i]->options());
    if (T > 0 && dys[0].defined()) {
      at::Tensor dy = dys[0].resolve_neg().contiguous();
      if (reinterpret_cast<uintptr_t>(dy.data_ptr()) % 4 != 0) dy = dy.clone(at::MemoryFormat::Contiguous);
      size_t bytes = 0;
      const at::Tensor ws = ffn_workspace(o.f, true, dy, &bytes);
      const float* g = saved[4].data_ptr<float>();
      auto out = [&](size_t i) { return grads[i].defined() ? grads[i].data_ptr() : nullptr; };
      entry_check(entries.ffn_backward(&o.f, o.x.data_ptr(), o.gate.data_ptr(), o.up.data_ptr(), o.down.data_ptr(), dy.data_ptr(), g, g + T * F,
                             out(0), out(1), out(2), out(3), ws.data_ptr(), bytes,
                             reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())),
                "came8_gated_ffn_backward");
    }
    if (again) {
      auto once = std::make_shared<torch::autograd::DelayedError>("gated_ffn is differentiable once", 4);
      torch::autograd::variable_list in(4);
      for (size_t i = 0; i < 4; ++i)
        if (grads[i].defined()) in[i] = grads[i].detach().set_requires_grad(true);
      at::AutoGradMode grad(true);
      auto marked = (*once)(std::move(in));
      for (size_t i = 0; i < 4; ++i)
        if (grads[i].defined()) grads[i] = marked[i];
    }
    return grads;
  }
};

// bind(*addresses): of libcame8's entries, in the order of Entries
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7])) return nullptr;
  auto take = [&](auto& entry, int i) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(a[i]); };
  take(entries.error, 0);
  take(entries.adamw, 1);
  take(entries.norm_size, 2);
  take(entries.norm, 3);
  take(entries.clip, 4);
  take(entries.ffn_size, 5);
  take(entries.ffn_forward, 6);
  take(entries.ffn_backward, 7);
  Py_RETURN_NONE;
}

// gated_ffn(x, w_gate, w_up, w_down, activation: int, stream: int) -> y
PyObject* gated_ffn(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* po[4];
  long long act, stream;
  if (!PyArg_ParseTuple(args, "OOOOLL", &po[0], &po[1], &po[2], &po[3], &act, &stream)) return nullptr;
  TORCH_CHECK(!torch::jit::tracer::isTracing(), "gated_ffn: cannot be traced; a trace would hold the result's allocation alone");
  const char* names[4] = {"x", "w_gate", "w_up", "w_down"};
  at::Tensor t[4];
  for (int i = 0; i < 4; ++i) {
    TORCH_CHECK(THPVariable_Check(po[i]), "gated_ffn: came_amd runs on the GPU; ", names[i], " is ", Py_TYPE(po[i])->tp_name);
    t[i] = THPVariable_Unpack(po[i]);
    // without an operand that needs a gradient no autograd node would refuse it, and the result would have no tangent
    TORCH_CHECK(!t[i]._fw_grad(0).defined(), "gated_ffn: no forward-mode derivatives; ", names[i], " has a tangent");
    TORCH_CHECK(t[i].is_cuda(), "gated_ffn: came_amd runs on the GPU; ", names[i], " is a ", t[i].device(), " tensor");
    TORCH_CHECK(t[i].layout() == at::kStrided && dtype_code(t[i]) >= 0, "gated_ffn: unsupported dtype ", dtype_name(t[i]), " of ",
                names[i], " (float32, bfloat16 and float16 are supported)");
    TORCH_CHECK(t[i].scalar_type() == t[0].scalar_type() && t[i].device() == t[0].device(), "gated_ffn: ", names[i], " is ",
                dtype_name(t[i]), " on ", t[i].device(), ", x is ", dtype_name(t[0]), " on ", t[0].device());
  }
  const at::Tensor &x = t[0], &gate = t[1], &up = t[2], &down = t[3];
  TORCH_CHECK_VALUE(x.dim() >= 1 && gate.dim() == 2 && up.sizes() == gate.sizes() && down.dim() == 2,
                    "gated_ffn: x [..., dim], w_gate and w_up [hidden, dim], w_down [out, hidden]; got ", x.sizes(), ", ",
                    gate.sizes(), ", ", up.sizes(), ", ", down.sizes());
  TORCH_CHECK_VALUE(x.size(-1) == gate.size(1) && down.size(1) == gate.size(0) && gate.numel() > 0 && down.numel() > 0,
                    "gated_ffn: widths do not match or are empty: ", x.sizes(), ", ", gate.sizes(), ", ", down.sizes());
  pybind11::gil_scoped_release no_gil;
  const int64_t tokens = x.numel() / x.size(-1);
  const at::Tensor rows = x.dim() == 2 ? x : x.reshape({tokens, x.size(-1)});
  at::Tensor y;
  if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || up.requires_grad() || down.requires_grad()))
    y = GatedFfn::apply(rows, gate, up, down, int64_t(act), int64_t(stream));
  else
    y = ffn_forward(rows, gate, up, down, act, stream, false).first;
  if (x.dim() != 2) {
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = down.size(0);
    y = y.view(sizes);
  }
  pybind11::gil_scoped_acquire gil;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"gather", gather, METH_VARARGS, "descriptors of a param group's tensors"},
                         {"adamw_step", adamw_step, METH_VARARGS, "one AdamW step of a param group"},
                         {"grad_norm", grad_norm, METH_VARARGS, "the norm of gradients, and the clip by it"},
                         {"bind", bind, METH_VARARGS, "libcame8's entries"},
                         {"gated_ffn", gated_ffn, METH_VARARGS, "the gated feed-forward block"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "came8_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_came8_host(void) { return PyModule_Create(&module); }
