// The gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T and its gradients: argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
#include <limits>
#include <type_traits>

#include "../../include/came8.h"
#include "came8_ffn.h"
#include "came8_ops.h"

namespace came8 {
namespace {

int64_t up(int64_t n, int64_t a) { return (n + a - 1) / a * a; }

// What lies in the workspace: h (and dg, du), and copies of the operands whose rows do not start on words or end inside a
// chunk (k_ffn_pack).  Every row there starts 16 bytes aligned and ends in zeros.
struct Layout {
  int64_t ldh = 0;  // elements
  size_t h = 0, dg = 0, du = 0, bytes = 0;
  struct Copy {
    int64_t ld = 0;  // 0: read where it is
    size_t at = 0;
  } x, gate, up, down, dy;
};

bool ragged(const came8_ffn* f, int64_t cols, int64_t ld) {
  return f->dtype == CAME8_F32 ? cols % 4 != 0 : cols % 8 != 0 || ld % 2 != 0;
}

Layout layout_of(const came8_ffn* f, bool backward) {
  Layout l;
  const int64_t es = f->dtype == CAME8_F32 ? 4 : 2;
  auto take = [&](int64_t rows, int64_t ld) {
    const size_t at = l.bytes;
    l.bytes += size_t(up(rows * ld * es, 256));
    return at;
  };
  auto copy = [&](Layout::Copy& c, int64_t rows, int64_t cols, int64_t ld) {
    if (!ragged(f, cols, ld)) return;
    c.ld = up(cols, 16 / es);
    c.at = take(rows, c.ld);
  };
  l.ldh = up(f->hidden, 16 / es);
  l.h = take(f->tokens, l.ldh);
  if (backward) {
    l.dg = take(f->tokens, l.ldh);
    l.du = take(f->tokens, l.ldh);
    copy(l.dy, f->tokens, f->out, f->out);
  }
  copy(l.x, f->tokens, f->dim, f->ld_x);
  copy(l.gate, f->hidden, f->dim, f->ld_gate);
  copy(l.up, f->hidden, f->dim, f->ld_up);
  copy(l.down, f->out, f->hidden, f->ld_down);
  return l;
}

// The operand as the kernels read it: itself, or its copy in the workspace.
template <typename S>
Operand operand(const void* p, int64_t rows, int64_t cols, int64_t ld, const Layout::Copy& c, char* ws, hipStream_t stream) {
  if (c.ld == 0) return {p, ld};
  hipLaunchKernelGGL(k_ffn_pack<S>, dim3(unsigned(std::min<int64_t>(rows, 1 << 16))), dim3(kThreads), 0, stream,
                     static_cast<const S*>(p), ld, reinterpret_cast<S*>(ws + c.at), c.ld, rows, int32_t(cols));
  return {ws + c.at, c.ld};
}

constexpr int64_t kMaxTokens = int64_t(1) << 24;
constexpr int64_t kMaxStride = int64_t(1) << 20;   // of rows, in elements: a tile's 256 rows stay below 2^31 bytes
constexpr int64_t kMaxMatrix = int64_t(1) << 36;   // elements: a launch's work items stay below 2^32

int check(const char* what, const came8_ffn* f) {
  const std::string at = std::string(what) + ": ";
  if (f == nullptr) return op_fail(CAME8_EINVAL, at + "no description given");
  if (f->dtype != CAME8_F32 && f->dtype != CAME8_BF16 && f->dtype != CAME8_F16)
    return op_fail(CAME8_EINVAL, at + "unknown dtype " + std::to_string(f->dtype));
  if (f->activation < CAME8_ACT_SILU || f->activation > CAME8_ACT_GELU_TANH)
    return op_fail(CAME8_EINVAL, at + "unknown activation " + std::to_string(f->activation));
  if (f->tokens < 0 || f->tokens > kMaxTokens || f->dim < 1 || f->hidden < 1 || f->out < 1 || f->out > kMaxStride)
    return op_fail(CAME8_EINVAL, at + "tokens must be in [0, 2^24], dim, hidden and out in [1, 2^20]");
  const int64_t strides[4][2] = {{f->ld_x, f->dim}, {f->ld_gate, f->dim}, {f->ld_up, f->dim}, {f->ld_down, f->hidden}};
  for (const auto& s : strides)
    if (s[0] < s[1] || s[0] > kMaxStride)
      return op_fail(CAME8_EINVAL, at + "a row stride must be at least the row's length and at most 2^20");
  for (const int64_t n : {f->tokens * f->hidden, f->tokens * f->out, f->tokens * f->dim, f->hidden * f->dim, f->hidden * f->out})
    if (n > kMaxMatrix) return op_fail(CAME8_EINVAL, at + "a matrix of more than 2^36 elements");
  return CAME8_OK;
}

int check_pointers(const char* what, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (p == nullptr || reinterpret_cast<uintptr_t>(p) % 4 != 0)
      return op_fail(CAME8_EINVAL, std::string(what) + ": a null pointer, or one that is not 4 bytes aligned");
  return CAME8_OK;
}

template <typename T, int B, int WAVES_N, bool AROWS, bool BROWS, Epilogue EPI>
bool launch_tiles(GemmArgs a, int64_t least, hipStream_t stream) {
  constexpr int cols = EPI == kGate ? B / 2 : B;
  a.tiles_m = (a.M + B - 1) / B;
  a.tiles_n = (a.N + cols - 1) / cols;
  const int64_t tiles = int64_t(a.tiles_m) * a.tiles_n;
  if (tiles < least) return false;
  hipLaunchKernelGGL((k_ffn_gemm<T, B, B, WAVES_N, AROWS, BROWS, EPI>), dim3(unsigned(tiles)), dim3(2 * WAVES_N * kWave), 0, stream, a);
  return true;
}

template <typename T, bool AROWS, bool BROWS, Epilogue EPI>
void launch(const GemmArgs& a, hipStream_t stream) {
#ifndef MIN256
#define MIN256 200
#endif
#ifndef MIN128
#define MIN128 200
#endif
  if constexpr (!std::is_same<T, F32>::value)
    if (launch_tiles<T, 256, 4, AROWS, BROWS, EPI>(a, MIN256, stream)) return;
  if (launch_tiles<T, 128, 2, AROWS, BROWS, EPI>(a, MIN128, stream)) return;
  launch_tiles<T, 64, 2, AROWS, BROWS, EPI>(a, 0, stream);
}

template <typename T>
void forward(const came8_ffn* f, const void* x, const void* wg, const void* wu, const void* wd, void* y, float* g, float* u,
             const Layout& l, char* ws, hipStream_t stream) {
  GemmArgs a{};
  a.nseg = 1;
  a.act = f->activation;
  a.M = int32_t(f->tokens), a.N = int32_t(f->hidden), a.K = int32_t(f->dim);
  a.seg[0] = {operand<typename T::storage>(x, f->tokens, f->dim, f->ld_x, l.x, ws, stream),
              operand<typename T::storage>(wg, f->hidden, f->dim, f->ld_gate, l.gate, ws, stream)};
  a.b2 = operand<typename T::storage>(wu, f->hidden, f->dim, f->ld_up, l.up, ws, stream);
  a.out = ws + l.h, a.ldo = l.ldh;
  a.g = g, a.u = u, a.ldg = f->hidden;
  launch<T, true, true, kGate>(a, stream);
  GemmArgs d{};
  d.nseg = 1;
  d.M = int32_t(f->tokens), d.N = int32_t(f->out), d.K = int32_t(f->hidden);
  d.seg[0] = {{ws + l.h, l.ldh}, operand<typename T::storage>(wd, f->out, f->hidden, f->ld_down, l.down, ws, stream)};
  d.out = y, d.ldo = f->out;
  launch<T, true, true, kStore>(d, stream);
}

template <typename T>
void backward(const came8_ffn* f, const void* x, const void* wg, const void* wu, const void* wd, const void* dy, const float* g,
              const float* u, void* dx, void* dwg, void* dwu, void* dwd, const Layout& l, char* ws, hipStream_t stream) {
  GemmArgs a{};
  a.nseg = 1;
  a.act = f->activation;
  a.M = int32_t(f->tokens), a.N = int32_t(f->hidden), a.K = int32_t(f->out);
  const Operand pdy = operand<typename T::storage>(dy, f->tokens, f->out, f->out, l.dy, ws, stream);
  const Operand px = operand<typename T::storage>(x, f->tokens, f->dim, f->ld_x, l.x, ws, stream);
  a.seg[0] = {pdy, operand<typename T::storage>(wd, f->out, f->hidden, f->ld_down, l.down, ws, stream)};
  a.out = ws + l.dg, a.out2 = ws + l.du, a.out3 = dwd ? ws + l.h : nullptr, a.ldo = l.ldh;
  a.g = const_cast<float*>(g), a.u = const_cast<float*>(u), a.ldg = f->hidden;
  launch<T, true, false, kBack>(a, stream);
  GemmArgs d{};
  if (dx) {
    d.nseg = 2;
    d.M = int32_t(f->tokens), d.N = int32_t(f->dim), d.K = int32_t(f->hidden);
    d.seg[0] = {{ws + l.dg, l.ldh}, operand<typename T::storage>(wg, f->hidden, f->dim, f->ld_gate, l.gate, ws, stream)};
    d.seg[1] = {{ws + l.du, l.ldh}, operand<typename T::storage>(wu, f->hidden, f->dim, f->ld_up, l.up, ws, stream)};
    d.out = dx, d.ldo = f->dim;
    launch<T, true, false, kStore>(d, stream);
  }
  d.nseg = 1;
  d.K = int32_t(f->tokens);
  d.M = int32_t(f->hidden), d.N = int32_t(f->dim), d.ldo = f->dim;
  if (dwg) {
    d.seg[0] = {{ws + l.dg, l.ldh}, px};
    d.out = dwg;
    launch<T, false, false, kStore>(d, stream);
  }
  if (dwu) {
    d.seg[0] = {{ws + l.du, l.ldh}, px};
    d.out = dwu;
    launch<T, false, false, kStore>(d, stream);
  }
  if (dwd) {
    d.M = int32_t(f->out), d.N = int32_t(f->hidden), d.ldo = f->hidden;
    d.seg[0] = {pdy, {ws + l.h, l.ldh}};
    d.out = dwd;
    launch<T, false, false, kStore>(d, stream);
  }
}

}  // namespace
}  // namespace came8

using namespace came8;

extern "C" {

int came8_gated_ffn_workspace_size(const came8_ffn* f, int32_t backward, size_t* bytes) {
  try {
    const int rc = check("came8_gated_ffn_workspace_size", f);
    if (rc != CAME8_OK) return rc;
    if (bytes == nullptr) return op_fail(CAME8_EINVAL, "came8_gated_ffn_workspace_size: bytes is NULL");
    *bytes = std::max<size_t>(layout_of(f, backward != 0).bytes, 256);
    return CAME8_OK;
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string("came8_gated_ffn_workspace_size: ") + e.what());
  }
}

int came8_gated_ffn_forward(const came8_ffn* f, const void* x, const void* w_gate, const void* w_up, const void* w_down, void* y,
                            float* g, float* u, void* workspace, size_t workspace_bytes, void* stream) {
  try {
    const char* what = "came8_gated_ffn_forward";
    int rc = check(what, f);
    if (rc != CAME8_OK) return rc;
    if (f->tokens == 0) return CAME8_OK;
    if ((rc = check_pointers(what, {x, w_gate, w_up, w_down, y})) != CAME8_OK) return rc;
    if ((g == nullptr) != (u == nullptr)) return op_fail(CAME8_EINVAL, std::string(what) + ": g and u are kept together");
    const Layout l = layout_of(f, false);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < l.bytes)
      return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
    char* ws = static_cast<char*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (f->dtype == CAME8_F32) forward<F32>(f, x, w_gate, w_up, w_down, y, g, u, l, ws, s);
    else if (f->dtype == CAME8_BF16) forward<BF16>(f, x, w_gate, w_up, w_down, y, g, u, l, ws, s);
    else forward<F16>(f, x, w_gate, w_up, w_down, y, g, u, l, ws, s);
    return op_check_launch("gated_ffn_forward");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string("came8_gated_ffn_forward: ") + e.what());
  }
}

int came8_gated_ffn_backward(const came8_ffn* f, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                             const void* dy, const float* g, const float* u, void* dx, void* dw_gate, void* dw_up,
                             void* dw_down, void* workspace, size_t workspace_bytes, void* stream) {
  try {
    const char* what = "came8_gated_ffn_backward";
    int rc = check(what, f);
    if (rc != CAME8_OK) return rc;
    if (f->tokens == 0) return op_fail(CAME8_EINVAL, std::string(what) + ": no tokens");
    if ((rc = check_pointers(what, {x, w_gate, w_up, w_down, dy})) != CAME8_OK) return rc;
    if (g == nullptr || u == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": null pointer");
    for (const void* p : {dx, dw_gate, dw_up, dw_down})
      if (p != nullptr && (rc = check_pointers(what, {p})) != CAME8_OK) return rc;
    const Layout l = layout_of(f, true);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < l.bytes)
      return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
    char* ws = static_cast<char*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (f->dtype == CAME8_F32) backward<F32>(f, x, w_gate, w_up, w_down, dy, g, u, dx, dw_gate, dw_up, dw_down, l, ws, s);
    else if (f->dtype == CAME8_BF16) backward<BF16>(f, x, w_gate, w_up, w_down, dy, g, u, dx, dw_gate, dw_up, dw_down, l, ws, s);
    else backward<F16>(f, x, w_gate, w_up, w_down, dy, g, u, dx, dw_gate, dw_up, dw_down, l, ws, s);
    return op_check_launch("gated_ffn_backward");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string("came8_gated_ffn_backward: ") + e.what());
  }
}

}  // extern "C"
