// AdamW over many tensors (fp32 or 8-bit moments), the global gradient norm and the clip by it.
//
// All of it is one pass over memory: per element a few multiply-adds against 10 to 28 bytes.  The kernels are
// multi-tensor: a table of up to 64 (192 for the norm) tensors travels in the kernel's arguments, a workgroup takes one
// chunk of one tensor and finds it by comparing its number with the table's chunk starts, one a lane.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <utility>
#include <vector>

#include "../../include/came8.h"
#include "came8_device.h"
#include "came8_ops.h"

namespace came8 {
namespace {

constexpr int kAdamTab = 64;    // tensors a launch: 60 bytes each of the 4 KB of arguments
constexpr int kGradTab = 192;   // 18 bytes each; a multiple of a wavefront's lanes (find_tensor)
// Elements of a workgroup: 256 lanes by 8 by 4 rows; a launch that has fewer than kSmallLaunch of those takes single rows (or
// as few as a block of 8-bit moments needs), since then only its latency counts: 192 adapters of 10 to 33 thousand elements,
// three launches of 11.2 us in 4 rows and of 7.4 in single ones.
constexpr int kAdamRow = 2048;
constexpr int kAdamRows = 4;
constexpr int kSmallLaunch = 512;
constexpr int kGradChunk = 16384;
constexpr int kNormGroups = 2048;  // workgroups of a norm launch: eight a CU, what is resident
constexpr float kTinyBlock = 0x1p-100f;  // 8-bit blocks whose largest is below hold zeros (127/a and 1.875/a stay finite)

struct AdamTab {
  void* p[kAdamTab];
  const void* g[kAdamTab];
  void* m[kAdamTab];
  void* v[kAdamTab];
  float* ma[kAdamTab];
  float* va[kAdamTab];
  int64_t n[kAdamTab];
  int32_t start[kAdamTab];  // first chunk
  int32_t count;
  float b1, c1, b2, c2, eps;
  float decay;      // 1 - lr * weight_decay
  float step_size;  // lr / (1 - beta1^t)
  float inv_bc2;    // 1 / sqrt(1 - beta2^t)
  uint32_t key;
  int32_t log2b;
  const float* scale;
};
static_assert(sizeof(AdamTab) <= 4096, "kernel arguments");

struct GradTab {
  void* g[kGradTab];
  uint32_t n_lo[kGradTab];
  int32_t start[kGradTab];
  uint16_t n_hi_dt[kGradTab];  // numel >> 32, and the type in the lowest two bits
  int32_t count;
  int32_t chunks;
};
static_assert(sizeof(GradTab) <= 4096, "kernel arguments");

// The table's entry that chunk c belongs to: starts ascend from 0, so it is the number of starts <= c, less one.
template <int N>
__device__ __forceinline__ int find_tensor(const int32_t (&start)[N], int count, int c) {
  const int lane = threadIdx.x & (kWave - 1);
  int k = 0;
#pragma unroll
  for (int i = 0; i < N; i += kWave)
    k += __popcll(__ballot(i + lane < count && start[i + lane] <= c));
  return __builtin_amdgcn_readfirstlane(k - 1);
}

template <size_t N>
struct BitsOf;
template <>
struct BitsOf<1> { using type = uint8_t; };
template <>
struct BitsOf<2> { using type = uint16_t; };
template <>
struct BitsOf<4> { using type = uint32_t; };
template <size_t N>
using Bits = typename BitsOf<N>::type;

// V consecutive elements at p[i] as the words they fill, those from n on as zeros; any address the type allows.  Streamed
// operands of at most 16 bytes a lane take the nontemporal hint.
template <typename T, int V>
struct Row {
  using storage = typename T::storage;
  static constexpr int kWords = V * int(sizeof(storage)) / 4;
  static constexpr bool kNt = kWords <= 4;
  typedef uint32_t raw __attribute__((ext_vector_type(kWords), aligned(sizeof(storage))));
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const CAME8_GLOBAL storage* p, int64_t i, int64_t n) {
    if (i + V <= n) {
      const CAME8_GLOBAL raw* a = (const CAME8_GLOBAL raw*)(p + i);
      const raw r = kNt ? __builtin_nontemporal_load(a) : *a;
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = r[k];
    } else {
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < n) {
          constexpr int per = 4 / int(sizeof(storage));
          w[e / per] |= uint32_t(__builtin_bit_cast(Bits<sizeof(storage)>, p[i + e])) << (32 / per * (e % per));
        }
    }
  }
  __device__ __forceinline__ void store(CAME8_GLOBAL storage* p, int64_t i, int64_t n) const {
    if (i + V <= n) {
      raw r;
#pragma unroll
      for (int k = 0; k < kWords; ++k) r[k] = w[k];
      CAME8_GLOBAL raw* a = (CAME8_GLOBAL raw*)(p + i);
      if (kNt) __builtin_nontemporal_store(r, a);
      else *a = r;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < n) {
          constexpr int per = 4 / int(sizeof(storage));
          p[i + e] = __builtin_bit_cast(storage, Bits<sizeof(storage)>(w[e / per] >> (32 / per * (e % per))));
        }
    }
  }
  __device__ __forceinline__ float get(int e) const { return T::elem(w, e); }
  __device__ __forceinline__ void put(const float (&in)[V]) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      if constexpr (sizeof(storage) == 4) w[k] = __float_as_uint(in[k]);
      else w[k] = uint32_t(T::store(in[2 * k])) | uint32_t(T::store(in[2 * k + 1])) << 16;
    }
  }
};
struct U8 {
  using storage = uint8_t;
};

// ---------------------------------------------------------------------------------------------- fp32 moments
// Bound by memory: 16 + 3 types' bytes an element, every load of 4 rounds issued before the first value is used.
// 355 M fp32 parameters and the norm before it 1970 us (5.8 TB/s), 1.07 G bf16 ones 4281 us (5.5 TB/s); one round at a time
// 2040 and 4420, eight elements a lane (two instructions an fp32 operand, each touching half of the lines) 2185 and 4650,
// without the nontemporal hint 2181 and 4550.  The divide and square root are the IEEE ones: the memory hides them.
template <typename P, typename G, int ROWS>
__global__ __launch_bounds__(kThreads) void k_adamw32(const AdamTab tab) {
  constexpr int V = 4, U = ROWS == 1 ? 2 : 4, kAdamChunk = kAdamRow * ROWS;
  const int t = find_tensor(tab.start, tab.count, int(blockIdx.x));
  const int64_t n = tab.n[t];
  const int64_t base = int64_t(int(blockIdx.x) - tab.start[t]) * kAdamChunk;
  auto* p = gbl(static_cast<typename P::storage*>(tab.p[t]));
  auto* g = gbl(static_cast<const typename G::storage*>(tab.g[t]));
  auto* m = gbl(static_cast<float*>(tab.m[t]));
  auto* v = gbl(static_cast<float*>(tab.v[t]));
  const float scale = tab.scale ? *tab.scale : 1.0f;
  for (int c = 0; c < kAdamChunk; c += kThreads * V * U) {
    if (base + c >= n) return;
    Row<G, V> gr[U];
    Row<P, V> pr[U];
    Row<F32, V> mr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = base + c + (u * kThreads + threadIdx.x) * V;
      gr[u].load(g, i, n);
      mr[u].load(m, i, n);
      vr[u].load(v, i, n);
      pr[u].load(p, i, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = base + c + (u * kThreads + threadIdx.x) * V;
      float pn[V], mn[V], vn[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = gr[u].get(e) * scale;
        mn[e] = mr[u].get(e) * tab.b1 + x * tab.c1;
        vn[e] = vr[u].get(e) * tab.b2 + (x * x) * tab.c2;
        pn[e] = pr[u].get(e) * tab.decay - tab.step_size * (mn[e] / (sqrtf(vn[e]) * tab.inv_bc2 + tab.eps));
      }
      mr[u].put(mn);
      vr[u].put(vn);
      pr[u].put(pn);
      mr[u].store(m, i, n);
      vr[u].store(v, i, n);
      pr[u].store(p, i, n);
    }
  }
}

// ----------------------------------------------------------------------------------------------- 8-bit moments
// The second moment's codes: y in [0, 1.875] times 2^-96 puts the format's grid (5 exponent, 3 fraction bits) on fp32's
// own, the format's subnormals on fp32's, so a code is the value's upper 12 bits and rounding adds below them.
constexpr float kSmall = 0x1p-96f, kLarge = 0x1p96f;

// 32 bits for a pair of elements, 16 to each
__device__ __forceinline__ uint32_t pair_hash(uint32_t pair, uint32_t key) {
  uint32_t x = (pair ^ key) * 0x9E3779B1u;
  x = (x ^ (x >> 15)) * 0x85EBCA77u;
  return x ^ (x >> 13);
}

// One wavefront takes 4 rows (or 1 or 2) of 512 elements, 8 to a lane; a block is a part of a row, a row (K = 1), or K rows, so its
// largest is a reduction over lanes and no LDS is used.  Bound by memory: 1.07 G bf16 parameters 1913 us, 5.6 TB/s of their
// 10 bytes each (1922 with one row loaded at a time), though some 60 operations an element come near what the vector units
// issue meanwhile; an IEEE square root and division would be over it.
template <typename P, typename G, int K, int ROWS>
__global__ __launch_bounds__(kThreads) void k_adamw8(const AdamTab tab) {
  constexpr int kAdamChunk = kAdamRow * ROWS;
  const int t = find_tensor(tab.start, tab.count, int(blockIdx.x));
  const int64_t n = tab.n[t];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int64_t base = int64_t(int(blockIdx.x) - tab.start[t]) * kAdamChunk + wave * (512 * ROWS) + lane * 8;
  auto* p = gbl(static_cast<typename P::storage*>(tab.p[t]));
  auto* g = gbl(static_cast<const typename G::storage*>(tab.g[t]));
  auto* mq = gbl(static_cast<uint8_t*>(tab.m[t]));
  auto* vq = gbl(static_cast<uint8_t*>(tab.v[t]));
  auto *ma = gbl(tab.ma[t]), *va = gbl(tab.va[t]);
  const float scale = tab.scale ? *tab.scale : 1.0f;
  const int lanes = K > 1 ? kWave : min(kWave, 1 << (tab.log2b - 3));  // of a block in a row
  constexpr int L = ROWS;  // loaded together
  Row<G, 8> gr[L];
  Row<P, 8> pr[L];
  Row<U8, 8> mc[L], vc[L];
  float sm[L], sv[L];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const int64_t i = base + l * 512;
    gr[l].load(g, i, n);
    mc[l].load(mq, i, n);
    vc[l].load(vq, i, n);
    pr[l].load(p, i, n);
    const int64_t b = i >> tab.log2b;
    sm[l] = i < n ? ma[b] : 0.0f;
    sv[l] = i < n ? va[b] : 0.0f;
  }
#pragma unroll
  for (int r0 = 0; r0 < L; r0 += K) {
    float m[K][8], v[K][8];
    uint32_t mtop = 0, vtop = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int l = r0 + k;
      const int64_t i = base + (r0 + k) * 512;
      const float fm = scale_s8(sm[l]), fv = sv[l] * float(8.0 / 15.0);
      float pn[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = gr[l].get(e) * scale;
        const uint32_t c = (vc[l].w[e >> 2] >> (8 * (e & 3))) & 255u;
        m[k][e] = (code_elem(mc[l].w, e) * fm) * tab.b1 + x * tab.c1;
        v[k][e] = ((__uint_as_float(c << 20) * kLarge) * fv) * tab.b2 + (x * x) * tab.c2;
        mtop = max(mtop, __float_as_uint(m[k][e]) & 0x7fffffffu);
        vtop = max(vtop, __float_as_uint(v[k][e]) & 0x7fffffffu);
        // hardware square root and reciprocal (an ulp each): p's update only, and the denominator is at least eps > 0
        const float d = __builtin_amdgcn_sqrtf(v[k][e]) * tab.inv_bc2 + tab.eps;
        pn[e] = pr[l].get(e) * tab.decay - tab.step_size * (m[k][e] * __builtin_amdgcn_rcpf(d));
      }
      pr[l].put(pn);
      pr[l].store(p, i, n);
    }
    // bits of non-negative floats order as they do, with infinities and then NaNs on top: a block keeps its NaN
    float am = __uint_as_float(group_max_bits_rt(mtop, lanes)), av = __uint_as_float(group_max_bits_rt(vtop, lanes));
    const float im = am < kTinyBlock ? 0.0f : 127.0f / am, iv = av < kTinyBlock ? 0.0f : 1.875f / av;
    if (am < kTinyBlock) am = 1.0f;
    if (av < kTinyBlock) av = 1.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t i = base + (r0 + k) * 512;
      if (i >= n) continue;
      Row<U8, 8> mn, vn;
      mn.w[0] = mn.w[1] = vn.w[0] = vn.w[1] = 0;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t h = pair_hash(uint32_t((i + e) >> 1), tab.key);
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int s = 8 * ((e + o) & 3);
          const float q = fminf(127.0f, fmaxf(-127.0f, rintf(m[k][e + o] * im)));
          mn.w[e >> 2] |= (uint32_t(int(q)) & 255u) << s;
          const uint32_t random = (o ? h >> 16 : h & 0xffffu) << 4 | 8u;
          const uint32_t bits = __float_as_uint((v[k][e + o] * iv) * kSmall) + random;
          vn.w[e >> 2] |= min(bits >> 20, 255u) << s;
        }
      }
      mn.store(mq, i, n);
      vn.store(vq, i, n);
      if (k == 0 && lane % lanes == 0) {
        const int64_t b = i >> tab.log2b;
        ma[b] = am;
        va[b] = av;
      }
    }
  }
}

// 4 rows of 4 consecutive codes a lane, all loaded before the first is used: five bytes an element, the memory's rate.
constexpr int kDequantTile = 4096;
__global__ __launch_bounds__(kThreads) void k_dequantize_e5m3(const uint8_t* q, const float* absmax, int64_t n, int32_t log2b,
                                                              float* out) {
  const int64_t ntiles = (n + kDequantTile - 1) / kDequantTile;
  for (int64_t tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
    const int64_t base = tile * kDequantTile + threadIdx.x * 4;
    uint32_t w[4] = {};
    float a[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = base + r * (kThreads * 4);
      if (i + 4 <= n) {
        w[r] = *(const CAME8_GLOBAL u32u*)(gbl(q) + i);
      } else {
        for (int e = 0; i + e < n; ++e) w[r] |= uint32_t(gbl(q)[i + e]) << (8 * e);
      }
      a[r] = i < n ? gbl(absmax)[i >> log2b] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = base + r * (kThreads * 4);
      const float s = a[r] * float(8.0 / 15.0);
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (__uint_as_float(((w[r] >> (8 * e)) & 255u) << 20) * kLarge) * s;
      if (i + 4 <= n) {
        __builtin_nontemporal_store(f32x4u{x[0], x[1], x[2], x[3]}, (CAME8_GLOBAL f32x4u*)(gbl(out) + i));
      } else {
        for (int e = 0; i + e < n; ++e) gbl(out)[i + e] = x[e];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------- norm and clip
// 16 bytes a lane
template <typename T>
constexpr int kLaneElems = 16 / int(sizeof(typename T::storage));

template <typename T>
__device__ __forceinline__ float sum_squares(const void* data, int64_t base, int64_t n) {
  constexpr int V = kLaneElems<T>, U = 8;
  auto* g = gbl(static_cast<const typename T::storage*>(data));
  float acc[V] = {};
  for (int c = 0; c < kGradChunk && base + c < n; c += kThreads * V * U) {
    Row<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(g, base + c + (u * kThreads + threadIdx.x) * V, n);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(x[u].get(e), x[u].get(e), acc[e]);
  }
#pragma unroll
  for (int s = V / 2; s > 0; s /= 2)
#pragma unroll
    for (int e = 0; e < s; ++e) acc[e] += acc[e + s];
  return acc[0];
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = wave_sum(v);
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// One fp64 partial per workgroup, at its own place.  Eight 16-byte loads a lane in flight: norm and scale of 0.4 G bf16
// gradients 395 us together (gradients of 0.8 GB: the scale's read comes from HBM again), 403 with four and two.
__global__ __launch_bounds__(kThreads) void k_grad_squares(const GradTab tab, double* partial) {
  __shared__ double lds[4];
  double acc = 0.0;
  for (int c = int(blockIdx.x); c < tab.chunks; c += int(gridDim.x)) {
    const int t = find_tensor(tab.start, tab.count, c);
    const int64_t n = int64_t(tab.n_lo[t]) | int64_t(tab.n_hi_dt[t] >> 2) << 32;
    const int64_t base = int64_t(c - tab.start[t]) * kGradChunk;
    switch (tab.n_hi_dt[t] & 3) {
      case CAME8_F32: acc += double(sum_squares<F32>(tab.g[t], base, n)); break;
      case CAME8_BF16: acc += double(sum_squares<BF16>(tab.g[t], base, n)); break;
      default: acc += double(sum_squares<F16>(tab.g[t], base, n)); break;
    }
  }
  acc = block_sum(acc, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// The partials' sum in the order of their places (the same bits whatever order they were written in), the norm and the
// clip's factor.  A launch of its own: the alternative, the last workgroup to arrive, needs a counter that is zero.
__global__ __launch_bounds__(kThreads) void k_grad_norm(const double* partial, int count, float max_norm, float* norm,
                                                        float* factor) {
  __shared__ double lds[4];
  double acc = 0.0;
  for (int i = int(threadIdx.x); i < count; i += kThreads) acc += partial[i];
  acc = block_sum(acc, lds);
  if (threadIdx.x != 0) return;
  const float nrm = float(sqrt(acc));
  *norm = nrm;
  if (factor == nullptr) return;
  const float f = max_norm / (nrm + 1e-6f);
  *factor = f > 1.0f ? 1.0f : f;  // a NaN stays
}

template <typename T>
__device__ __forceinline__ void scale_chunk(void* data, int64_t base, int64_t n, float f) {
  constexpr int V = kLaneElems<T>, U = 4;
  auto* g = gbl(static_cast<typename T::storage*>(data));
  for (int c = 0; c < kGradChunk && base + c < n; c += kThreads * V * U) {
    Row<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(g, base + c + (u * kThreads + threadIdx.x) * V, n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = x[u].get(e) * f;
      x[u].put(y);
      x[u].store(g, base + c + (u * kThreads + threadIdx.x) * V, n);
    }
  }
}

__global__ __launch_bounds__(kThreads) void k_grad_scale(const GradTab tab, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int c = int(blockIdx.x); c < tab.chunks; c += int(gridDim.x)) {
    const int t = find_tensor(tab.start, tab.count, c);
    const int64_t n = int64_t(tab.n_lo[t]) | int64_t(tab.n_hi_dt[t] >> 2) << 32;
    const int64_t base = int64_t(c - tab.start[t]) * kGradChunk;
    switch (tab.n_hi_dt[t] & 3) {
      case CAME8_F32: scale_chunk<F32>(tab.g[t], base, n, f); break;
      case CAME8_BF16: scale_chunk<BF16>(tab.g[t], base, n, f); break;
      default: scale_chunk<F16>(tab.g[t], base, n, f); break;
    }
  }
}

// ------------------------------------------------------------------------------------------------------ host
int64_t chunks_of(int64_t n, int64_t chunk) { return (n + chunk - 1) / chunk; }
bool type_ok(int32_t dt) { return dt == CAME8_F32 || dt == CAME8_BF16 || dt == CAME8_F16; }
size_t size_of(int32_t dt) { return dt == CAME8_F32 ? 4 : 2; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int64_t kMaxElements = int64_t(1) << 36;  // of a tensor; 192 tensors' chunks stay below 2^31
constexpr int64_t kMaxGroups = int64_t(1) << 23;    // of a launch: its work items stay below 2^32

using AdamFn = void (*)(AdamTab);

// rows: in and out, how many a workgroup's wavefronts take; 1 asks for the fewest that the block size allows
template <typename P, typename G>
AdamFn adam_kernel(int bits, int block, int& rows) {
  if (bits == 32) return rows == 1 ? k_adamw32<P, G, 1> : k_adamw32<P, G, kAdamRows>;
  if (block == 2048) rows = 4;
  if (block == 1024 && rows == 1) rows = 2;
  if (block == 2048) return k_adamw8<P, G, 4, 4>;
  if (block == 1024) return rows == 2 ? k_adamw8<P, G, 2, 2> : k_adamw8<P, G, 2, 4>;
  return rows == 1 ? k_adamw8<P, G, 1, 1> : k_adamw8<P, G, 1, 4>;
}
template <typename P>
AdamFn adam_kernel_g(int gdt, int bits, int block, int& rows) {
  return gdt == CAME8_F32 ? adam_kernel<P, F32>(bits, block, rows)
         : gdt == CAME8_BF16 ? adam_kernel<P, BF16>(bits, block, rows) : adam_kernel<P, F16>(bits, block, rows);
}
AdamFn adam_kernel_of(int pdt, int gdt, int bits, int block, int& rows) {
  return pdt == CAME8_F32 ? adam_kernel_g<F32>(gdt, bits, block, rows)
         : pdt == CAME8_BF16 ? adam_kernel_g<BF16>(gdt, bits, block, rows) : adam_kernel_g<F16>(gdt, bits, block, rows);
}

uint32_t mix(uint32_t x) {
  x *= 0x9E3779B1u;
  x = (x ^ (x >> 15)) * 0x85EBCA77u;
  return x ^ (x >> 13);
}

int refuse(const char* what, int32_t tensor, const char* why) {
  return op_fail(CAME8_EINVAL, std::string(what) + ": tensor " + std::to_string(tensor) + ": " + why);
}

int check_grads(const char* what, const came8_grad_tensor* ts, int32_t n) {
  if (n < 0 || (n > 0 && ts == nullptr)) return op_fail(CAME8_EINVAL, std::string(what) + ": no tensors given");
  for (int32_t i = 0; i < n; ++i) {
    const came8_grad_tensor& t = ts[i];
    if (!type_ok(t.dtype)) return refuse(what, i, "unknown dtype");
    if (t.numel < 0 || t.numel > kMaxElements) return refuse(what, i, "bad numel");
    if (t.numel > 0 && (t.data == nullptr || !aligned(t.data, size_of(t.dtype)))) return refuse(what, i, "null or misaligned pointer");
  }
  return CAME8_OK;
}

// The tables of a tensor list, empty tensors left out.
std::vector<GradTab> grad_tables(const came8_grad_tensor* ts, int32_t n) {
  std::vector<GradTab> out;
  for (int32_t i = 0; i < n; ++i) {
    if (ts[i].numel == 0) continue;
    const int64_t chunks = chunks_of(ts[i].numel, kGradChunk);
    if (out.empty() || out.back().count == kGradTab) {
      out.emplace_back();
      out.back().count = out.back().chunks = 0;
    }
    GradTab& t = out.back();
    const int k = t.count++;
    t.g[k] = ts[i].data;
    t.n_lo[k] = uint32_t(ts[i].numel);
    t.n_hi_dt[k] = uint16_t(uint64_t(ts[i].numel) >> 32 << 2 | uint64_t(ts[i].dtype));
    t.start[k] = t.chunks;
    t.chunks += int32_t(chunks);
  }
  return out;
}

// Whether some tensors have memory in common (one that is listed twice).  Lists in the order of their addresses, as the views of
// a flat buffer, or against it, are told without sorting (192 tensors: 1 us).
bool share_memory(const came8_grad_tensor* ts, int32_t n) {
  using Range = std::pair<uintptr_t, uintptr_t>;  // first byte, end
  auto range = [](const came8_grad_tensor& t) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.data);
    return Range(p, p + uintptr_t(t.numel) * size_of(t.dtype));
  };
  bool up = true, down = true;
  Range last(0, 0);
  bool any = false;
  for (int32_t i = 0; i < n && (up || down); ++i) {
    if (ts[i].numel == 0) continue;
    const Range r = range(ts[i]);
    if (any) {
      up = up && r.first >= last.second;
      down = down && r.second <= last.first;
    }
    any = true;
    last = r;
  }
  if (up || down) return false;
  std::vector<Range> at;
  at.reserve(size_t(n));
  for (int32_t i = 0; i < n; ++i)
    if (ts[i].numel > 0) at.push_back(range(ts[i]));
  std::sort(at.begin(), at.end());
  for (size_t i = 1; i < at.size(); ++i)
    if (at[i].first < at[i - 1].second) return true;  // of sorted ones, some two neighbours overlap if any two do
  return false;
}

int grad_norm(const char* what, const std::vector<GradTab>& tabs, int32_t n, double max_norm, float* norm, float* factor,
              void* workspace, size_t bytes, hipStream_t stream) {
  if (norm == nullptr || workspace == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": null pointer");
  if (!(max_norm >= 0.0)) return op_fail(CAME8_EINVAL, std::string(what) + ": max_norm must be >= 0");
  if (bytes < came8_grad_norm_workspace_size(n) || !aligned(workspace, 8))
    return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
  double* partial = static_cast<double*>(workspace);
  int total = 0;
  for (const GradTab& t : tabs) {
    const int groups = std::min(t.chunks, kNormGroups);
    hipLaunchKernelGGL(k_grad_squares, dim3(groups), dim3(kThreads), 0, stream, t, partial + total);
    total += groups;
  }
  hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kThreads), 0, stream, partial, total, float(max_norm), norm, factor);
  return op_check_launch("grad_norm");
}

}  // namespace
}  // namespace came8

using namespace came8;

extern "C" {

size_t came8_grad_norm_workspace_size(int32_t n_tensors) {
  const size_t launches = n_tensors <= 0 ? 1 : (size_t(n_tensors) + kGradTab - 1) / kGradTab;
  return launches * kNormGroups * sizeof(double);
}

int came8_grad_norm(const came8_grad_tensor* tensors, int32_t n_tensors, double max_norm, float* norm, float* factor,
                    void* workspace, size_t workspace_bytes, void* stream) {
  try {
    const int rc = check_grads("came8_grad_norm", tensors, n_tensors);
    if (rc != CAME8_OK) return rc;
    return grad_norm("came8_grad_norm", grad_tables(tensors, n_tensors), n_tensors, max_norm, norm, factor, workspace,
                     workspace_bytes, static_cast<hipStream_t>(stream));
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string("came8_grad_norm: ") + e.what());
  }
}

int came8_grad_clip(const came8_grad_tensor* tensors, int32_t n_tensors, double max_norm, float* norm, float* factor,
                    void* workspace, size_t workspace_bytes, void* stream) {
  try {
    int rc = check_grads("came8_grad_clip", tensors, n_tensors);
    if (rc != CAME8_OK) return rc;
    if (factor == nullptr) return op_fail(CAME8_EINVAL, "came8_grad_clip: null pointer");
    const std::vector<GradTab> tabs = grad_tables(tensors, n_tensors);
    rc = grad_norm("came8_grad_clip", tabs, n_tensors, max_norm, norm, factor, workspace, workspace_bytes,
                   static_cast<hipStream_t>(stream));
    if (rc != CAME8_OK) return rc;
    auto scale = [&](const std::vector<GradTab>& some) {
      for (const GradTab& t : some)
        hipLaunchKernelGGL(k_grad_scale, dim3(unsigned(std::min<int64_t>(t.chunks, kMaxGroups))), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), t, factor);
    };
    if (!share_memory(tensors, n_tensors)) {
      scale(tabs);
    } else {  // launches one after another, or two workgroups would scale the same values
      for (int32_t i = 0; i < n_tensors; ++i) scale(grad_tables(tensors + i, 1));
    }
    return op_check_launch("grad_scale");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string("came8_grad_clip: ") + e.what());
  }
}

int came8_adamw_step(const came8_adamw_tensor* tensors, int32_t n_tensors, const came8_adamw_hparams* hp,
                     const float* grad_scale, void* stream) {
  try {
    if (hp == nullptr || n_tensors < 0 || (n_tensors > 0 && tensors == nullptr))
      return op_fail(CAME8_EINVAL, "came8_adamw_step: no tensors or hyper-parameters given");
    if (hp->bits != 32 && hp->bits != 8) return op_fail(CAME8_EINVAL, "came8_adamw_step: bits must be 32 or 8");
    const int B = hp->block_size;
    if (hp->bits == 8 && (B < 64 || B > 2048 || (B & (B - 1)) != 0))
      return op_fail(CAME8_EINVAL, "came8_adamw_step: block_size must be a power of two in [64, 2048]");
    if (!(hp->lr >= 0.0) || !(hp->beta1 >= 0.0 && hp->beta1 < 1.0) || !(hp->beta2 >= 0.0 && hp->beta2 < 1.0) ||
        !(hp->eps >= 0.0) || !(hp->weight_decay >= 0.0))
      return op_fail(CAME8_EINVAL, "came8_adamw_step: lr, eps and weight_decay must be >= 0, betas in [0, 1)");
    if (hp->bits == 8 && !(float(hp->eps) >= std::numeric_limits<float>::min()))
      return op_fail(CAME8_EINVAL, "came8_adamw_step: 8-bit moments need eps > 0 (a normal fp32 number)");
    if (hp->flags != 0) return op_fail(CAME8_EINVAL, "came8_adamw_step: unknown flags");
    for (int32_t i = 0; i < n_tensors; ++i) {
      const came8_adamw_tensor& t = tensors[i];
      const char* what = "came8_adamw_step";
      if (!type_ok(t.param_dtype) || !type_ok(t.grad_dtype)) return refuse(what, i, "unknown dtype");
      if (t.numel < 0 || t.numel > kMaxElements) return refuse(what, i, "bad numel");
      if (t.step < 1) return refuse(what, i, "step must be >= 1");
      if (t.numel == 0) continue;
      const size_t ms = hp->bits == 32 ? 4 : 1;
      if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || !aligned(t.param, size_of(t.param_dtype)) ||
          !aligned(t.grad, size_of(t.grad_dtype)) || !aligned(t.exp_avg, ms) || !aligned(t.exp_avg_sq, ms))
        return refuse(what, i, "null or misaligned pointer");
      if (hp->bits == 8 && (!t.exp_avg_absmax || !t.exp_avg_sq_absmax || !aligned(t.exp_avg_absmax, 4) ||
                            !aligned(t.exp_avg_sq_absmax, 4)))
        return refuse(what, i, "null or misaligned absmax");
    }
    // launches: tensors of one (types, step count) together, in the order given
    std::vector<char> done(size_t(n_tensors), 0);
    for (int32_t i = 0; i < n_tensors; ++i) {
      if (done[size_t(i)] || tensors[i].numel == 0) continue;
      const came8_adamw_tensor& f = tensors[i];
      AdamTab tab;
      const double t = double(f.step);
      tab.b1 = float(hp->beta1);
      tab.c1 = float(1.0 - hp->beta1);
      tab.b2 = float(hp->beta2);
      tab.c2 = float(1.0 - hp->beta2);
      tab.eps = float(hp->eps);
      tab.decay = float(1.0 - hp->lr * hp->weight_decay);
      tab.step_size = float(hp->lr / (1.0 - std::pow(hp->beta1, t)));
      tab.inv_bc2 = float(1.0 / std::sqrt(1.0 - std::pow(hp->beta2, t)));
      tab.key = mix(mix(hp->seed) ^ uint32_t(f.step));
      tab.log2b = hp->bits == 8 ? __builtin_ctz(unsigned(B)) : 0;
      tab.scale = grad_scale;
      int64_t chunks = 0;  // of kAdamRows rows
      tab.count = 0;
      auto flush = [&]() {
        if (tab.count == 0) return;
        int rows = chunks < kSmallLaunch ? 1 : kAdamRows;
        const AdamFn fn = adam_kernel_of(f.param_dtype, f.grad_dtype, hp->bits, B, rows);
        int64_t groups = 0;
        for (int k = 0; k < tab.count; ++k) {
          tab.start[k] = int32_t(groups);
          groups += chunks_of(tab.n[k], int64_t(kAdamRow) * rows);
        }
        hipLaunchKernelGGL(fn, dim3(unsigned(groups)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), tab);
        tab.count = 0;
        chunks = 0;
      };
      for (int32_t j = i; j < n_tensors; ++j) {
        const came8_adamw_tensor& a = tensors[j];
        if (done[size_t(j)] || a.numel == 0 || a.step != f.step || a.param_dtype != f.param_dtype || a.grad_dtype != f.grad_dtype)
          continue;
        done[size_t(j)] = 1;
        const int64_t c = chunks_of(a.numel, int64_t(kAdamRow) * kAdamRows);
        if (tab.count == kAdamTab || chunks + c > kMaxGroups) flush();
        const int k = tab.count++;
        tab.p[k] = a.param;
        tab.g[k] = a.grad;
        tab.m[k] = a.exp_avg;
        tab.v[k] = a.exp_avg_sq;
        tab.ma[k] = a.exp_avg_absmax;
        tab.va[k] = a.exp_avg_sq_absmax;
        tab.n[k] = a.numel;
        chunks += c;
      }
      flush();
    }
    return op_check_launch("adamw_step");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string("came8_adamw_step: ") + e.what());
  }
}

int came8_dequantize_second_moment(const uint8_t* q, const float* absmax, int64_t n, int32_t block_size, float* out,
                                   void* stream) {
  if (block_size < 64 || block_size > 2048 || (block_size & (block_size - 1)) != 0)
    return op_fail(CAME8_EINVAL, "came8_dequantize_second_moment: block_size must be a power of two in [64, 2048]");
  if (n < 0) return op_fail(CAME8_EINVAL, "came8_dequantize_second_moment: n must be >= 0");
  if (n == 0) return CAME8_OK;
  if (!q || !absmax || !out) return op_fail(CAME8_EINVAL, "came8_dequantize_second_moment: null pointer");
  hipLaunchKernelGGL(k_dequantize_e5m3, dim3(unsigned(std::min<int64_t>(chunks_of(n, kDequantTile), kMaxGroups))),
                     dim3(kThreads), 0, static_cast<hipStream_t>(stream), q, absmax, n, __builtin_ctz(unsigned(block_size)), out);
  return op_check_launch("dequantize_second_moment");
}

}  // extern "C"
