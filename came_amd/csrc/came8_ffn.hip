// The gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T and its gradients: argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
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
  size_t h = 0, dg = 0, du = 0, part = 0, bytes = 0;
  struct Copy {
    int64_t ld = 0;  // 0: read where it is
    size_t at = 0;
  } x, gate, up, down, dy;
};

bool ragged(const came8_ffn* f, int64_t cols, int64_t ld) {
  return f->dtype == CAME8_F32 ? cols % 4 != 0 : cols % 8 != 0 || ld % 2 != 0;
}

// How a product is cut: tiles of `tile` by `tile` (fp32 at 256: 128 wide; gate and up: half as many columns of h), `splits`
// workgroups a tile.
struct Cut {
  int tile = 0, splits = 1;
};
struct Size {
  int64_t M, N, K;
  int nseg;
};
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int width_of(bool fp32, int tile) { return fp32 && tile == 256 ? 128 : tile; }

// What a tile size runs at: workgroups at once on the GPU, and a step of k (128 bytes) of one, microseconds.
struct Speed {
  int tile, at_once;
  double half, full;  // 16-bit types, fp32
};
constexpr Speed kSpeeds[] = {{256, 256, 1.87, 3.3}, {128, 512, 1.22, 3.8}, {64, 1024, 1.19, 1.9}};
constexpr int kSplitSteps = 4;   // a share of a sum has at least these steps
constexpr int kMaxSplits = 8;    // 32 tokens of 4096 and 11008 68.4 us with 16, 65.8 with 8, 70.5 with 4; 64 tokens 82.1, 77.8, 81.5
constexpr double kJoinBytes = 4e6;  // a microsecond of k_ffn_join: shares written and read

int64_t steps_of(const came8_ffn* f, const Size& z) { return ceil_div(z.K, f->dtype == CAME8_F32 ? 32 : 64) * z.nseg; }

// The cut with the least estimated time: rounds of workgroups by their steps, and three more for the first loads and the
// epilogue, and what joining the shares moves.
Cut cut_of(const came8_ffn* f, const Size& z, bool gate) {
  Cut best;
  double least = 1e300;
  for (const Speed& v : kSpeeds) {
    const double us = f->dtype == CAME8_F32 ? v.full : v.half;
    const int width = width_of(f->dtype == CAME8_F32, v.tile);
    const int64_t tiles = ceil_div(z.M, v.tile) * ceil_div(z.N, gate ? width / 2 : width), steps = steps_of(f, z);
    for (int s = 1; s <= kMaxSplits; ++s) {
      if (s > 1 && steps / s < kSplitSteps) break;
      const double t = double(ceil_div(tiles * s, v.at_once)) * (double(ceil_div(steps, s)) + 3.0) * us +
                       (s > 1 ? 4.0 + double(s) * double(z.M) * double(z.N) * (gate ? 16.0 : 8.0) / kJoinBytes : 0.0);
      if (t < least) {
        least = t;
        best.tile = v.tile;
        best.splits = s;
      }
    }
  }
  return best;
}

// The cuts of several products in one launch: one tile size, the one whose tiles keep the GPU busy for the least time; a
// product whose sums are longer than an even share of all work is split.
void cut_together(const came8_ffn* f, const Size* z, int count, Cut* cuts) {
  double least = 1e300;
  for (const Speed& v : kSpeeds) {
    const double us = f->dtype == CAME8_F32 ? v.full : v.half;
    const int width = width_of(f->dtype == CAME8_F32, v.tile);
    double work = 0.0, join = 0.0;
    int64_t longest = 0;
    for (int i = 0; i < count; ++i)
      work += double(ceil_div(z[i].M, v.tile) * ceil_div(z[i].N, width)) * (double(steps_of(f, z[i])) + 3.0);
    const int64_t share = std::max<int64_t>(2 * kSplitSteps, int64_t(work / v.at_once));
    int splits[4];
    for (int i = 0; i < count; ++i) {
      const int64_t steps = steps_of(f, z[i]);
      splits[i] = int(std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, ceil_div(steps, share), steps / kSplitSteps})));
      longest = std::max(longest, ceil_div(steps, splits[i]) + 3);
      if (splits[i] > 1) join += double(splits[i]) * double(z[i].M) * double(z[i].N) * 8.0 / kJoinBytes;
    }
    if (join > 0.0) join += 4.0;
    const double t = (std::max(work / v.at_once, double(longest)) + 0.5 * double(longest)) * us + join;
    if (t < least) {
      least = t;
      for (int i = 0; i < count; ++i) cuts[i].tile = v.tile, cuts[i].splits = splits[i];
    }
  }
}

struct Cuts {
  Cut gate, down;          // forward
  Cut back, grads[4];      // backward: dh; dx, dw_gate, dw_up, dw_down
};
Cuts cuts_of(const came8_ffn* f) {
  Cuts c;
  c.gate = cut_of(f, {f->tokens, f->hidden, f->dim, 1}, true);
  c.down = cut_of(f, {f->tokens, f->out, f->hidden, 1}, false);
  c.back = cut_of(f, {f->tokens, f->hidden, f->out, 1}, false);
  const Size z[4] = {{f->tokens, f->dim, f->hidden, 2}, {f->hidden, f->dim, f->tokens, 1}, {f->hidden, f->dim, f->tokens, 1},
                     {f->out, f->hidden, f->tokens, 1}};
  cut_together(f, z, 4, c.grads);
  return c;
}

// Whether the forward product reads an odd-strided w_down where it is (Stage: ODD) instead of a copy of it: in tiles up to
// 128, where a copy would cost as much as the product (48 tokens of 2048 and 5461 in fp16 38.9 us with a copy, 31.7 without);
// tiles of 256 have no registers for it, and the copy is little beside them.
bool shifted_in_place(const came8_ffn* f) {
  return f->dtype != CAME8_F32 && f->ld_down % 2 != 0 && cuts_of(f).down.tile < 256;
}

int64_t part_floats(const Cut& c, int64_t M, int64_t N) { return c.splits > 1 ? c.splits * M * up(N, 4) : 0; }

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
  if (!backward && f->tokens <= kFewRows) {  // h in fp32
    l.h = take(f->tokens * 4 / es, l.ldh);
    return l;
  }
  l.h = take(f->tokens, l.ldh);
  if (backward) {
    l.dg = take(f->tokens, l.ldh);
    l.du = take(f->tokens, l.ldh);
    copy(l.dy, f->tokens, f->out, f->out);
  }
  copy(l.x, f->tokens, f->dim, f->ld_x);
  copy(l.gate, f->hidden, f->dim, f->ld_gate);
  copy(l.up, f->hidden, f->dim, f->ld_up);
  if (backward || !shifted_in_place(f)) copy(l.down, f->out, f->hidden, f->ld_down);
  // shares of split sums; dh's are joined before the others are written
  const Cuts c = cuts_of(f);
  int64_t part = std::max(2 * part_floats(c.gate, f->tokens, f->hidden), part_floats(c.down, f->tokens, f->out));
  if (backward)
    part = std::max(part_floats(c.back, f->tokens, f->hidden),
                    part_floats(c.grads[0], f->tokens, f->dim) + part_floats(c.grads[1], f->hidden, f->dim) +
                        part_floats(c.grads[2], f->hidden, f->dim) + part_floats(c.grads[3], f->out, f->hidden));
  l.part = l.bytes;
  l.bytes += size_t(up(part * 4, 256));
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

template <typename T>
void tile(GemmArgs& a, const Cut& c, bool gate) {
  const int width = width_of(std::is_same<T, F32>::value, c.tile), cols = gate ? width / 2 : width;
  a.tiles_m = int32_t(ceil_div(a.M, c.tile));
  a.tiles_n = int32_t(ceil_div(a.N, cols));
  a.splits = c.splits;
}

unsigned join_groups(const GemmArgs& a) {
  return unsigned(std::min<int64_t>(ceil_div(int64_t(a.M) * ((a.N + 3) / 4), kThreads), 1 << 14));
}

// One product over its tiles.  odd: the second operand's rows are an odd number of elements apart (shifted_in_place).
template <typename T, bool BROWS, Epilogue EPI>
void launch(GemmArgs a, const Cut& c, float* part, hipStream_t stream, bool odd = false) {
  tile<T>(a, c, EPI == kGate);
  a.part = c.splits > 1 ? part : nullptr;
  const dim3 grid(unsigned(a.tiles_m) * unsigned(a.tiles_n) * unsigned(a.splits));
  constexpr int kWide = std::is_same<T, F32>::value ? 2 : 4;
  if (c.tile == 256) hipLaunchKernelGGL((k_ffn_gemm<T, 256, kWide, true, BROWS, EPI, false>), grid, dim3(512), 0, stream, a);
  if constexpr (!std::is_same<T, F32>::value) {
    if constexpr (BROWS && EPI == kStore) {
      if (c.tile == 128 && odd) hipLaunchKernelGGL((k_ffn_gemm<T, 128, 2, true, true, kStore, true>), grid, dim3(256), 0, stream, a);
      if (c.tile == 64 && odd) hipLaunchKernelGGL((k_ffn_gemm<T, 64, 2, true, true, kStore, true>), grid, dim3(256), 0, stream, a);
    }
  }
  if (c.tile == 128 && !odd) hipLaunchKernelGGL((k_ffn_gemm<T, 128, 2, true, BROWS, EPI, false>), grid, dim3(256), 0, stream, a);
  if (c.tile == 64 && !odd) hipLaunchKernelGGL((k_ffn_gemm<T, 64, 2, true, BROWS, EPI, false>), grid, dim3(256), 0, stream, a);
  if (a.part) hipLaunchKernelGGL((k_ffn_join<T, EPI>), dim3(join_groups(a)), dim3(kThreads), 0, stream, a);
}

template <typename T>
void forward_few(const came8_ffn* f, const void* x, const void* wg, const void* wu, const void* wd, void* y, float* g, float* u,
                 const Layout& l, char* ws, hipStream_t stream) {
  FewArgs a{};
  a.x = x, a.ldx = f->ld_x;
  a.w[0] = wg, a.w[1] = wu, a.ldw[0] = f->ld_gate, a.ldw[1] = f->ld_up;
  a.M = int32_t(f->tokens), a.N = int32_t(f->hidden), a.K = int32_t(f->dim), a.act = f->activation;
  a.out = ws + l.h, a.ldo = l.ldh;
  a.g = g, a.u = u, a.ldg = f->hidden;
  hipLaunchKernelGGL((k_ffn_few<T, true>), dim3(unsigned(ceil_div(a.N, 16))), dim3(512), 0, stream, a);
  FewArgs d{};
  d.x = ws + l.h, d.ldx = l.ldh;
  d.w[0] = wd, d.ldw[0] = f->ld_down;
  d.M = int32_t(f->tokens), d.N = int32_t(f->out), d.K = int32_t(f->hidden);
  d.out = y, d.ldo = f->out;
  hipLaunchKernelGGL((k_ffn_few<T, false>), dim3(unsigned(ceil_div(d.N, 16))), dim3(512), 0, stream, d);
}

template <typename T>
void forward(const came8_ffn* f, const void* x, const void* wg, const void* wu, const void* wd, void* y, float* g, float* u,
             const Layout& l, char* ws, hipStream_t stream) {
  if (f->tokens <= kFewRows) return forward_few<T>(f, x, wg, wu, wd, y, g, u, l, ws, stream);
  GemmArgs a{};
  a.nseg = 1;
  a.act = f->activation;
  a.M = int32_t(f->tokens), a.N = int32_t(f->hidden), a.K = int32_t(f->dim);
  a.seg[0] = {operand<typename T::storage>(x, f->tokens, f->dim, f->ld_x, l.x, ws, stream),
              operand<typename T::storage>(wg, f->hidden, f->dim, f->ld_gate, l.gate, ws, stream)};
  a.b2 = operand<typename T::storage>(wu, f->hidden, f->dim, f->ld_up, l.up, ws, stream);
  a.out = ws + l.h, a.ldo = l.ldh;
  a.g = g, a.u = u, a.ldg = f->hidden;
  const Cuts c = cuts_of(f);
  float* part = reinterpret_cast<float*>(ws + l.part);
  launch<T, true, kGate>(a, c.gate, part, stream);
  GemmArgs d{};
  d.nseg = 1;
  d.M = int32_t(f->tokens), d.N = int32_t(f->out), d.K = int32_t(f->hidden);
  d.seg[0] = {{ws + l.h, l.ldh}, operand<typename T::storage>(wd, f->out, f->hidden, f->ld_down, l.down, ws, stream)};
  d.out = y, d.ldo = f->out;
  launch<T, true, kStore>(d, c.down, part, stream, shifted_in_place(f));
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
  const Cuts c = cuts_of(f);
  float* part = reinterpret_cast<float*>(ws + l.part);
  launch<T, false, kBack>(a, c.back, part, stream);

  GradArgs r{};
  int32_t groups = 0, count = 0;
  auto add = [&](GemmArgs& g, const Cut& cut, int64_t M, int64_t N, int64_t K, void* out) {
    g.nseg = std::max(g.nseg, 1);
    g.M = int32_t(M), g.N = int32_t(N), g.K = int32_t(K);
    g.out = out, g.ldo = N;
    tile<T>(g, cut, false);
    if (cut.splits > 1) {
      g.part = part;
      part += part_floats(cut, M, N);
    }
    groups += g.tiles_m * g.tiles_n * g.splits;
  };
  if (dx) {
    r.dx.nseg = 2;
    r.dx.seg[0] = {{ws + l.dg, l.ldh}, operand<typename T::storage>(wg, f->hidden, f->dim, f->ld_gate, l.gate, ws, stream)};
    r.dx.seg[1] = {{ws + l.du, l.ldh}, operand<typename T::storage>(wu, f->hidden, f->dim, f->ld_up, l.up, ws, stream)};
    add(r.dx, c.grads[0], f->tokens, f->dim, f->hidden, dx);
  }
  auto add_dw = [&](const Cut& cut, int64_t M, int64_t N, void* out, const Operand& first, const Operand& second) {
    if (out == nullptr) return;
    r.first[count] = groups;
    GemmArgs& g = r.dw[count++];
    g.seg[0] = {first, second};
    add(g, cut, M, N, f->tokens, out);
  };
  add_dw(c.grads[1], f->hidden, f->dim, dwg, {ws + l.dg, l.ldh}, px);
  add_dw(c.grads[2], f->hidden, f->dim, dwu, {ws + l.du, l.ldh}, px);
  add_dw(c.grads[3], f->out, f->hidden, dwd, pdy, {ws + l.h, l.ldh});
  for (int k = count; k < 4; ++k) r.first[k] = groups;
  if (groups == 0) return;
  const int t = c.grads[0].tile;
  constexpr int kWide = std::is_same<T, F32>::value ? 2 : 4;
  if (t == 256) hipLaunchKernelGGL((k_ffn_grads<T, 256, kWide>), dim3(unsigned(groups)), dim3(512), 0, stream, r);
  if (t == 128) hipLaunchKernelGGL((k_ffn_grads<T, 128, 2>), dim3(unsigned(groups)), dim3(256), 0, stream, r);
  if (t == 64) hipLaunchKernelGGL((k_ffn_grads<T, 64, 2>), dim3(unsigned(groups)), dim3(256), 0, stream, r);
  unsigned most = 0;
  for (const GemmArgs* g : {&r.dx, &r.dw[0], &r.dw[1], &r.dw[2]})
    if (g->part) most = std::max(most, join_groups(*g));
  if (most > 0) hipLaunchKernelGGL(k_ffn_join_grads<T>, dim3(most, 4), dim3(kThreads), 0, stream, r);
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
