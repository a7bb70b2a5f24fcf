// What the translation units of came8_host share: libcame8's entries and the checks of tensors.
#pragma once

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>

#include <string>

#include "../../include/came8.h"

namespace came8_host {

// libcame8's entries, which Python has loaded; pointers in the order of bind()'s arguments
struct Entries {
  decltype(&came8_last_error) error = nullptr;
  decltype(&came8_adamw_step) adamw = nullptr;
  decltype(&came8_grad_norm_workspace_size) norm_size = nullptr;
  decltype(&came8_grad_norm) norm = nullptr;
  decltype(&came8_grad_clip) clip = nullptr;
  decltype(&came8_gated_ffn_workspace_size) ffn_size = nullptr;
  decltype(&came8_gated_ffn_forward) ffn_forward = nullptr;
  decltype(&came8_gated_ffn_backward) ffn_backward = nullptr;
  decltype(&came8_embedding_forward) embedding_forward = nullptr;
  decltype(&came8_embedding_workspace_size) embedding_size = nullptr;
  decltype(&came8_embedding_backward) embedding_backward = nullptr;
  decltype(&came8_rms_norm_forward) rms_forward = nullptr;
  decltype(&came8_rms_norm_workspace_size) rms_size = nullptr;
  decltype(&came8_rms_norm_backward) rms_backward = nullptr;
  decltype(&came8_rms_norm_int8) rms_int8 = nullptr;
  decltype(&came8_quantize_rows) quantize_rows = nullptr;
  decltype(&came8_int8_linear_workspace_size) int8_size = nullptr;
  decltype(&came8_int8_linear_forward) int8_forward = nullptr;
  decltype(&came8_log_probs_workspace_size) logprob_size = nullptr;
  decltype(&came8_log_probs_forward) logprob_forward = nullptr;
  decltype(&came8_log_probs_backward) logprob_backward = nullptr;
};
extern Entries entries;

void entry_check(int rc, const char* what);

// CAME8_F32, CAME8_BF16 or CAME8_F16; -1 for another type
int dtype_code(const at::Tensor& t);
std::string dtype_name(const at::Tensor& t);

// The gradients, marked so that a gradient of one of them raises
torch::autograd::variable_list differentiable_once(torch::autograd::variable_list grads, const char* what);

// A leaf's gradient is accumulated on the stream that was current when the first living graph of the leaf was made.  Where that
// was outside of a capture, accumulating during one waits across streams that the capture does not have, on a thread of the
// engine's that has no one to raise to.  So a node raises before it comes to that, unless the other stream is captured too.
// `captured`: the node's forward pass was.
void check_captured(bool captured, const char* op, const at::Device& device);

PyObject* embedding(PyObject*, PyObject* args);
PyObject* rms_norm(PyObject*, PyObject* args);
PyObject* rms_norm_int8(PyObject*, PyObject* args);
PyObject* quantize_rows(PyObject*, PyObject* args);
PyObject* int8_linear(PyObject*, PyObject* args);
PyObject* token_log_probs(PyObject*, PyObject* args);

}  // namespace came8_host
