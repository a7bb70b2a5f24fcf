// The root-mean-square norm with the residual's addition, its gradients, and rows in 8 bits with a scale each.
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   g = dy w,  dx = r (g - h r^2 mean(g h)) + dh,  dw = sum over the rows of dy h r
//
// (r^2 is taken as two factors: without eps, of rows of 1e-20 say, it is no float32.)
//
// A row lies in the registers of the threads that share it from its one read on: 16 lanes, a wavefront, 256 threads or 1024, by
// its width.  All of it is bound by memory; widths that fit no registers are read again.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <type_traits>

#include "../../include/came8.h"
#include "came8_codes.h"
#include "came8_ops.h"
#include "came8_rms_grid.h"
#include "came8_rows.h"

namespace came8 {
namespace {

enum Output { kNormed, kNormed8, kRows8 };

struct RmsArgs {
  const void* x;
  const void* residual;  // or null
  const void* w;
  void* y;               // kNormed
  void* h;               // where there is a residual
  int8_t* q;             // kNormed8, kRows8
  float* scale;
  int64_t rows, D, ld_x, ld_r, ld_q;
  float eps;
};

// ------------------------------------------------------------------------------------------------- 8 bits
// A code is p * 127 / a rounded to nearest even, with a the largest |p| of the row: what the norm multiplies the row by moves
// none.  In fp32, p * (127 / a) is off by at most 4 roundings of 127, 3.1e-5 of a code; a value that is so near to a border
// between two is taken again from p and a in 64 bits, which hold both: from their quotient where p has 24 bits at most (16-bit
// types, rows as they are), since that is a tie or further from one than its rounding, and by nearest_code where p has 48 (8192 x
// 4096 with the residual 83 us with either; in 16 bits the quotient takes 39 and 44, nearest_code 42 and 48).
constexpr float kTiny = 0x1p-100f;  // the largest of a row below holds zeros: 127 / it may be infinite
constexpr float kBorder = 0.5f - 4e-5f;

// what a chunk's codes are made from: p of each value as its factors
template <int V>
struct Factors {
  float h[V], w[V];
};

// a row's largest |p| as bits of a double, exact, and 127 over it; inv 0: codes of zero
struct Largest {
  uint64_t bits;
  float inv;
  __device__ __forceinline__ explicit Largest(uint64_t b) : bits(b) {
    const float a = value();
    inv = a >= kTiny && a <= 0x1.fffffep127f ? 127.0f / a : 0.0f;
  }
  __device__ __forceinline__ float value() const { return float(__builtin_bit_cast(double, bits)); }
  // a r / 127; an infinity or NaN stays
  __device__ __forceinline__ float scale(float r) const { return value() < kTiny ? 0.0f : value() * r / 127.0f; }
};

__device__ __forceinline__ uint64_t magnitude(double p) { return __builtin_bit_cast(uint64_t, p) & 0x7fffffffffffffffull; }

// WIDE: products of two float32 values
template <int V, bool WIDE>
__device__ __forceinline__ void store_codes(int8_t* row, int64_t e0, int64_t D, const Factors<V>& f, const Largest& a) {
  if (e0 >= ((D + 15) & ~int64_t(15))) return;
  float c[V];
  bool near = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float x = f.h[v] * f.w[v] * a.inv;
    c[v] = rintf(x);
    near |= fabsf(x - c[v]) > kBorder;
  }
  if (near) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const double p = double(f.h[v]) * double(f.w[v]), top = __builtin_bit_cast(double, a.bits);
      if constexpr (WIDE) c[v] = nearest_code(f.h[v] * f.w[v] * a.inv, c[v], p, top);
      else c[v] = float(__builtin_rint(p * 127.0 / top));
    }
  }
  uint32_t w[V / 4];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int32_t code = a.inv > 0.0f ? int32_t(c[v]) : 0;  // past D h is 0
    w[v / 4] = (v % 4 ? w[v / 4] : 0u) | (uint32_t(code) & 0xffu) << (8 * (v % 4));
  }
  CAME8_GLOBAL uint32_t* p = (CAME8_GLOBAL uint32_t*)gbl(row + e0);
  if constexpr (V == 8) *(CAME8_GLOBAL u32x2*)p = u32x2{w[0], w[1]};
  else *p = w[0];
}

// The largest |p| of a thread's chunks, as bits of a double.  Where p is exact in fp32 (16-bit types, rows as they are) that of
// the fp32 products.
template <typename T, bool NORM>
struct Top {
  static constexpr bool kWide = NORM && sizeof(typename T::storage) == 4;
  typename std::conditional<kWide, uint64_t, uint32_t>::type bits = 0;
  __device__ __forceinline__ void add(float h, float w) {
    if constexpr (kWide) bits = max(bits, magnitude(double(h) * double(w)));
    else bits = max(bits, __float_as_uint(h * w) & 0x7fffffffu);
  }
  template <int TPR>
  __device__ __forceinline__ Largest of_row(uint32_t* lds) const {  // lds: 2 * TPR / 64 words
    if constexpr (kWide) return Largest(row_max64<TPR>(bits, lds));
    else return Largest(magnitude(double(__uint_as_float(row_max<TPR>(bits, lds)))));
  }
};

// TPR threads a row, NV chunks a thread
template <typename T, int TPR, int NV, Output OUT>
__global__ __launch_bounds__(TPR < kThreads ? kThreads : TPR) void k_rms(const RmsArgs a) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>, kBlock = TPR < kThreads ? kThreads : TPR, kRows = kBlock / TPR;
  __shared__ __attribute__((aligned(8))) float lds[2][4 * (TPR / kWave + 1)];
  const int t = int(threadIdx.x) % TPR;
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * kRows + int(threadIdx.x) / TPR; row < a.rows; row += int64_t(gridDim.x) * kRows, turn ^= 1) {
    u32x4 raw[NV], res[NV], wr[NV];
    const S* x = static_cast<const S*>(a.x) + row * a.ld_x;
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = load_raw<T>(x, int64_t(i * TPR + t) * V, a.D);
    if (OUT != kRows8 && a.residual != nullptr) {
      const S* r = static_cast<const S*>(a.residual) + row * a.ld_r;
#pragma unroll
      for (int i = 0; i < NV; ++i) res[i] = load_raw<T>(r, int64_t(i * TPR + t) * V, a.D);
    }
    if constexpr (OUT != kRows8) {
#pragma unroll
      for (int i = 0; i < NV; ++i) wr[i] = load_raw<T>(static_cast<const S*>(a.w), int64_t(i * TPR + t) * V, a.D);
    }
    float v[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack<T>(raw[i], v[i]);
    float r = 1.0f;
    if constexpr (OUT != kRows8) {
      if (a.residual != nullptr) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float b[V];
          unpack<T>(res[i], b);
#pragma unroll
          for (int e = 0; e < V; ++e) v[i][e] += b[e];
          const u32x4 h = pack<T>(v[i]);
          unpack<T>(h, v[i]);
          store_raw<T>(static_cast<S*>(a.h) + row * a.D, int64_t(i * TPR + t) * V, a.D, h);
        }
      }
      float s[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] = fmaf(v[i][e], v[i][e], s[0]);
      row_sum<TPR>(s, lds[turn]);
      r = 1.0f / sqrtf(s[0] / float(a.D) + a.eps);
    }
    if constexpr (OUT == kNormed) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float w[V];
        unpack<T>(wr[i], w);
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = v[i][e] * r * w[e];
        store_chunk<T>(static_cast<S*>(a.y) + row * a.D, int64_t(i * TPR + t) * V, a.D, v[i]);
      }
    } else {
      auto factors = [&](int i) {
        Factors<V> f;
#pragma unroll
        for (int e = 0; e < V; ++e) f.h[e] = v[i][e];
        if constexpr (OUT == kNormed8) {
          unpack<T>(wr[i], f.w);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) f.w[e] = 1.0f;
        }
        return f;
      };
      Top<T, OUT == kNormed8> top;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Factors<V> f = factors(i);
#pragma unroll
        for (int e = 0; e < V; ++e) top.add(f.h[e], f.w[e]);
      }
      const Largest most = top.template of_row<TPR>(reinterpret_cast<uint32_t*>(lds[turn] + 2 * (TPR / kWave + 1)));
      if (t == 0) gbl(a.scale)[row] = most.scale(r);
#pragma unroll
      for (int i = 0; i < NV; ++i) store_codes<V, Top<T, OUT == kNormed8>::kWide>(a.q + row * a.ld_q, int64_t(i * TPR + t) * V, a.D, factors(i), most);
    }
  }
}

// Rows of any width, a workgroup each: they are read for every pass over them.
template <typename T, Output OUT>
__global__ __launch_bounds__(1024) void k_rms_long(const RmsArgs a) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>, kTpr = 1024;
  __shared__ __attribute__((aligned(8))) float lds[2][4 * (kTpr / kWave + 1)];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const S* x = static_cast<const S*>(a.x) + row * a.ld_x;
    const S* r = a.residual ? static_cast<const S*>(a.residual) + row * a.ld_r : nullptr;
    const S* w = static_cast<const S*>(a.w);
    auto value = [&](int64_t e0, float(&v)[V], bool write) {
      load_chunk<T>(x, e0, a.D, v);
      if (OUT != kRows8 && r != nullptr) {
        float b[V];
        load_chunk<T>(r, e0, a.D, b);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += b[e];
        const u32x4 h = pack<T>(v);
        unpack<T>(h, v);
        if (write) store_raw<T>(static_cast<S*>(a.h) + row * a.D, e0, a.D, h);
      }
    };
    float rr = 1.0f;
    if constexpr (OUT != kRows8) {
      float s[1] = {0.0f};
      for (int64_t e0 = int64_t(threadIdx.x) * V; e0 < a.D; e0 += kTpr * V) {
        float v[V];
        value(e0, v, false);
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) part = fmaf(v[e], v[e], part);
        s[0] += part;
      }
      row_sum<kTpr>(s, lds[turn]);
      rr = 1.0f / sqrtf(s[0] / float(a.D) + a.eps);
    }
    auto factors = [&](int64_t e0, bool write) {
      Factors<V> f;
      value(e0, f.h, write);
      if constexpr (OUT != kRows8) {
        load_chunk<T>(w, e0, a.D, f.w);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f.w[e] = 1.0f;
      }
      return f;
    };
    if constexpr (OUT == kNormed) {
      for (int64_t e0 = int64_t(threadIdx.x) * V; e0 < a.D; e0 += kTpr * V) {
        Factors<V> f = factors(e0, true);
#pragma unroll
        for (int e = 0; e < V; ++e) f.h[e] = f.h[e] * rr * f.w[e];
        store_chunk<T>(static_cast<S*>(a.y) + row * a.D, e0, a.D, f.h);
      }
    } else {
      Top<T, OUT == kNormed8> top;
      for (int64_t e0 = int64_t(threadIdx.x) * V; e0 < a.D; e0 += kTpr * V) {
        const Factors<V> f = factors(e0, false);
#pragma unroll
        for (int e = 0; e < V; ++e) top.add(f.h[e], f.w[e]);
      }
      const Largest most = top.template of_row<kTpr>(reinterpret_cast<uint32_t*>(lds[turn] + 2 * (kTpr / kWave + 1)));
      if (threadIdx.x == 0) gbl(a.scale)[row] = most.scale(rr);
      // up to the next multiple of 16 codes, whose chunks past D hold zeros
      for (int64_t e0 = int64_t(threadIdx.x) * V; e0 < ((a.D + 15) & ~int64_t(15)); e0 += kTpr * V)
        store_codes<V, Top<T, OUT == kNormed8>::kWide>(a.q + row * a.ld_q, e0, a.D, factors(e0, true), most);
    }
  }
}

// --------------------------------------------------------------------------------------------------- gradients
struct RmsBackArgs {
  const void* h;
  const void* w;
  const void* dy;
  const void* dh;  // or null
  void* dx;        // or null
  float* part;     // dw's partial sums, [gridDim.x][D], or null
  int64_t rows, D, ld;
  float eps;
};

// A workgroup takes every gridDim.x-th row (or group of rows) and keeps its part of dw in registers.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR < kThreads ? kThreads : TPR) void k_rms_back(const RmsBackArgs a) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>, kBlock = TPR < kThreads ? kThreads : TPR, kRows = kBlock / TPR;
  __shared__ float lds[2][2 * (TPR / kWave + 1)];
  __shared__ float sums[kRows > 1 ? kRows * TPR * NV * V : 1];
  const int t = int(threadIdx.x) % TPR, group = int(threadIdx.x) / TPR;
  float dw[NV][V] = {};
  u32x4 wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) wr[i] = load_raw<T>(static_cast<const S*>(a.w), int64_t(i * TPR + t) * V, a.D);
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * kRows + group; row < a.rows; row += int64_t(gridDim.x) * kRows, turn ^= 1) {
    u32x4 hr[NV], gr[NV], er[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) hr[i] = load_raw<T>(static_cast<const S*>(a.h) + row * a.ld, int64_t(i * TPR + t) * V, a.D);
#pragma unroll
    for (int i = 0; i < NV; ++i) gr[i] = load_raw<T>(static_cast<const S*>(a.dy) + row * a.D, int64_t(i * TPR + t) * V, a.D);
    if (a.dh != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) er[i] = load_raw<T>(static_cast<const S*>(a.dh) + row * a.D, int64_t(i * TPR + t) * V, a.D);
    }
    float s[2] = {0.0f, 0.0f};  // sums of h^2 and g h
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float h[V], g[V], w[V];
      unpack<T>(hr[i], h);
      unpack<T>(gr[i], g);
      unpack<T>(wr[i], w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s[0] = fmaf(h[e], h[e], s[0]);
        s[1] = fmaf(g[e] * w[e], h[e], s[1]);
      }
    }
    row_sum<TPR>(s, lds[turn]);
    const float r = 1.0f / sqrtf(s[0] / float(a.D) + a.eps), c = r * (r * (s[1] / float(a.D)));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float h[V], g[V], w[V], d[V];
      unpack<T>(hr[i], h);
      unpack<T>(gr[i], g);
      unpack<T>(wr[i], w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dw[i][e] = fmaf(g[e], h[e] * r, dw[i][e]);
        d[e] = r * fmaf(-h[e], c, g[e] * w[e]);
      }
      if (a.dx != nullptr) {
        if (a.dh != nullptr) {
          float b[V];
          unpack<T>(er[i], b);
#pragma unroll
          for (int e = 0; e < V; ++e) d[e] += b[e];
        }
        store_chunk<T>(static_cast<S*>(a.dx) + row * a.D, int64_t(i * TPR + t) * V, a.D, d);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + int64_t(blockIdx.x) * a.D;
  if constexpr (kRows > 1) {
    constexpr int kRow = TPR * NV * V;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) sums[group * kRow + (i * TPR + t) * V + e] = dw[i][e];
    __syncthreads();
    for (int e = int(threadIdx.x); e < kRow && e < a.D; e += kBlock) {
      float v = sums[e];
      for (int k = 1; k < kRows; ++k) v += sums[k * kRow + e];
      gbl(part)[e] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t e0 = int64_t(i * TPR + t) * V;
#pragma unroll
      for (int e = 0; e < V; e += 4) store_chunk<F32>(part, e0 + e, a.D, {dw[i][e], dw[i][e + 1], dw[i][e + 2], dw[i][e + 3]});
    }
  }
}

// Rows of any width: dx of a row a workgroup (COLUMNS false); dw of 1024 chunks of columns from r of every row, which it takes
// from `scale` (COLUMNS true).
template <typename T, bool COLUMNS>
__global__ __launch_bounds__(1024) void k_rms_back_long(const RmsBackArgs a, float* inverse) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>, kTpr = 1024;
  if constexpr (COLUMNS) {
    // blockIdx.x: columns, blockIdx.y: every gridDim.y-th row
    const int64_t e0 = (int64_t(blockIdx.x) * kTpr + threadIdx.x) * V;
    float dw[V] = {};
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
      float h[V], g[V];
      load_chunk<T>(static_cast<const S*>(a.h) + row * a.ld, e0, a.D, h);
      load_chunk<T>(static_cast<const S*>(a.dy) + row * a.D, e0, a.D, g);
      const float r = gbl(inverse)[row];
#pragma unroll
      for (int e = 0; e < V; ++e) dw[e] = fmaf(g[e], h[e] * r, dw[e]);
    }
#pragma unroll
    for (int e = 0; e < V; e += 4)
      store_chunk<F32>(a.part + int64_t(blockIdx.y) * a.D, e0 + e, a.D, {dw[e], dw[e + 1], dw[e + 2], dw[e + 3]});
  } else {
    __shared__ float lds[2][2 * (kTpr / kWave + 1)];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
      float s[2] = {0.0f, 0.0f};
      for (int64_t e0 = int64_t(threadIdx.x) * V; e0 < a.D; e0 += kTpr * V) {
        float h[V], g[V], w[V];
        load_chunk<T>(static_cast<const S*>(a.h) + row * a.ld, e0, a.D, h);
        load_chunk<T>(static_cast<const S*>(a.dy) + row * a.D, e0, a.D, g);
        load_chunk<T>(static_cast<const S*>(a.w), e0, a.D, w);
        float p = 0.0f, q = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          p = fmaf(h[e], h[e], p);
          q = fmaf(g[e] * w[e], h[e], q);
        }
        s[0] += p;
        s[1] += q;
      }
      row_sum<kTpr>(s, lds[turn]);
      const float r = 1.0f / sqrtf(s[0] / float(a.D) + a.eps), c = r * (r * (s[1] / float(a.D)));
      if (threadIdx.x == 0 && inverse != nullptr) gbl(inverse)[row] = r;
      if (a.dx == nullptr) continue;
      for (int64_t e0 = int64_t(threadIdx.x) * V; e0 < a.D; e0 += kTpr * V) {
        float h[V], g[V], w[V], d[V];
        load_chunk<T>(static_cast<const S*>(a.h) + row * a.ld, e0, a.D, h);
        load_chunk<T>(static_cast<const S*>(a.dy) + row * a.D, e0, a.D, g);
        load_chunk<T>(static_cast<const S*>(a.w), e0, a.D, w);
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = r * fmaf(-h[e], c, g[e] * w[e]);
        if (a.dh != nullptr) {
          float b[V];
          load_chunk<T>(static_cast<const S*>(a.dh) + row * a.D, e0, a.D, b);
#pragma unroll
          for (int e = 0; e < V; ++e) d[e] += b[e];
        }
        store_chunk<T>(static_cast<S*>(a.dx) + row * a.D, e0, a.D, d);
      }
    }
  }
}

// dw of 32 columns: the sum of the partial sums' rows, 128 of them at a time (8 lanes of 4 columns each).
template <typename T>
__global__ __launch_bounds__(1024) void k_rms_join(const float* part, int32_t parts, int64_t D, void* dw) {
  __shared__ float lds[16][kRmsJoinColumns];
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
  for (int64_t c0 = int64_t(blockIdx.x) * kRmsJoinColumns; c0 < D; c0 += int64_t(gridDim.x) * kRmsJoinColumns) {
    const int64_t c = c0 + lane % 8 * 4;
    float v[4] = {};
#pragma unroll 4
    for (int r = wave * 8 + lane / 8; r < parts; r += 128) {
      float p[4];
      load_chunk<F32>(part + int64_t(r) * D, c, D, p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int o = 8; o < kWave; o *= 2) v[e] += __shfl_xor(v[e], o, kWave);
      if (lane < 8) lds[wave][lane * 4 + e] = v[e];
    }
    __syncthreads();
    const int64_t col = c0 + int(threadIdx.x);
    if (threadIdx.x < kRmsJoinColumns && col < D) {
      float s = lds[0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < 16; ++w) s += lds[w][threadIdx.x];
      gbl(static_cast<typename T::storage*>(dw))[col] = T::store(s);
    }
    __syncthreads();  // before the next columns' sums
  }
}

// ------------------------------------------------------------------------------------------------------ launches
constexpr int64_t kMaxParts = 512;       // workgroups that share dw's sum

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool is_long(const came8_rms_norm* n) { return n->dim > 16384; }

// Calls f with the threads a row and chunks a thread of width D.  Fewer threads than a row has chunks would read it in turns,
// more would idle; with more than 16 elements a thread 1024 threads have no registers for the backward pass's row and its part of dw.
template <typename T, typename F>
void by_width(int64_t D, F&& f) {
  constexpr int V = kChunk<T>;
  using std::integral_constant;
  if (D <= 16 * V) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (D <= 64 * V) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (D <= 128 * V) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (D <= 256 * V) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (D <= 512 * V) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (D <= 1024 * V) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 16 / V>{});  // 16384 elements
}

template <typename T, Output OUT>
void forward(const came8_rms_norm* n, const RmsArgs& a, hipStream_t stream) {
  if (is_long(n)) {
    hipLaunchKernelGGL((k_rms_long<T, OUT>), dim3(unsigned(rms_row_groups(n->rows, 1))), dim3(1024), 0, stream, a);
    return;
  }
  by_width<T>(n->dim, [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, kBlock = TPR < kThreads ? kThreads : TPR;
    hipLaunchKernelGGL((k_rms<T, TPR, NV, OUT>), dim3(unsigned(rms_row_groups(n->rows, kBlock / TPR))), dim3(kBlock), 0, stream, a);
  });
}

template <Output OUT>
void forward_of(const came8_rms_norm* n, const RmsArgs& a, hipStream_t stream) {
  if (n->dtype == CAME8_F32) forward<F32, OUT>(n, a, stream);
  else if (n->dtype == CAME8_BF16) forward<BF16, OUT>(n, a, stream);
  else forward<F16, OUT>(n, a, stream);
}

// workgroups of the backward kernel
int64_t parts_of(const came8_rms_norm* n) {
  const int64_t V = n->dtype == CAME8_F32 ? 4 : 8, rows = n->dim <= 16 * V ? 16 : n->dim <= 256 * V ? 4 : 1;
  return std::min(ceil_div(n->rows, rows), is_long(n) ? 64 : kMaxParts);
}

template <typename T>
void backward(const came8_rms_norm* n, RmsBackArgs a, void* dw, void* ws, hipStream_t stream) {
  const int64_t parts = parts_of(n);
  a.part = dw ? static_cast<float*>(ws) : nullptr;
  if (is_long(n)) {
    float* inverse = dw ? a.part + parts * n->dim : nullptr;
    hipLaunchKernelGGL((k_rms_back_long<T, false>), dim3(unsigned(rms_row_groups(n->rows, 1))), dim3(1024), 0, stream, a, inverse);
    if (dw)
      hipLaunchKernelGGL((k_rms_back_long<T, true>), dim3(unsigned(rms_column_groups(n->dim, kChunk<T>)), unsigned(parts)), dim3(1024), 0,
                         stream, a, inverse);
  } else {
    by_width<T>(n->dim, [&](auto tpr, auto nv) {
      constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, kBlock = TPR < kThreads ? kThreads : TPR;
      hipLaunchKernelGGL((k_rms_back<T, TPR, NV>), dim3(unsigned(parts)), dim3(kBlock), 0, stream, a);
    });
  }
  if (dw)
    hipLaunchKernelGGL(k_rms_join<T>, dim3(unsigned(rms_join_groups(n->dim))), dim3(1024), 0, stream, a.part, int32_t(parts), n->dim, dw);
}

int check(const char* what, const came8_rms_norm* n, bool residual) {
  const std::string at = std::string(what) + ": ";
  if (n == nullptr) return op_fail(CAME8_EINVAL, at + "no description given");
  if (n->dtype != CAME8_F32 && n->dtype != CAME8_BF16 && n->dtype != CAME8_F16)
    return op_fail(CAME8_EINVAL, at + "unknown dtype " + std::to_string(n->dtype));
  if (n->rows < 0 || n->rows >= (int64_t(1) << 31) || n->dim < 1 || n->dim > kRmsMaxDim)
    return op_fail(CAME8_EINVAL, at + "rows must be in [0, 2^31), dim in [1, 2^30]");
  if (n->ld_x < n->dim || (residual && n->ld_residual < n->dim))
    return op_fail(CAME8_EINVAL, at + "a row stride must be at least the row's length");
  if (n->ld_x > (int64_t(1) << 31) || n->ld_residual > (int64_t(1) << 31))
    return op_fail(CAME8_EINVAL, at + "a row stride must be at most 2^31");
  return CAME8_OK;
}

int check_eps(const char* what, const came8_rms_norm* n) {
  if (std::isfinite(n->eps) && n->eps >= 0.0 && std::isfinite(float(n->eps))) return CAME8_OK;
  return op_fail(CAME8_EINVAL, std::string(what) + ": eps must be finite, in float32 too, and at least 0");
}
// in float32; above 0 where eps is, so that a row of zeros is not divided by it
float eps_of(const came8_rms_norm* n) {
  const float e = float(n->eps);
  return n->eps > 0.0 ? std::max(e, std::numeric_limits<float>::denorm_min()) : e;
}

// every pointer is there and aligned to its elements
int check_pointers(const char* what, int32_t dtype, std::initializer_list<const void*> ps) {
  const uintptr_t size = dtype == CAME8_F32 ? 4 : 2;
  for (const void* p : ps)
    if (p == nullptr || reinterpret_cast<uintptr_t>(p) % size != 0)
      return op_fail(CAME8_EINVAL, std::string(what) + ": a null pointer, or one that is not aligned to its type");
  return CAME8_OK;
}

int check_codes(const char* what, const came8_rms_norm* n, const int8_t* q, int64_t ld_q, const float* scale) {
  if (q == nullptr || reinterpret_cast<uintptr_t>(q) % 16 != 0 || ld_q % 16 != 0 || ld_q < n->dim || ld_q > (int64_t(1) << 31))
    return op_fail(CAME8_EINVAL, std::string(what) + ": rows of q start at multiples of 16 bytes and hold dim codes");
  return check_pointers(what, CAME8_F32, {scale});
}

}  // namespace
}  // namespace came8

using namespace came8;

extern "C" {

int came8_rms_norm_forward(const came8_rms_norm* n, const void* x, const void* residual, const void* weight, void* y, void* h,
                           void* stream) {
  const char* what = "came8_rms_norm_forward";
  try {
    int rc = check(what, n, residual != nullptr);
    if (rc != CAME8_OK || (rc = check_eps(what, n)) != CAME8_OK) return rc;
    if (n->rows == 0) return CAME8_OK;
    if ((rc = check_pointers(what, n->dtype, {x, weight, y})) != CAME8_OK) return rc;
    if ((residual == nullptr) != (h == nullptr)) return op_fail(CAME8_EINVAL, std::string(what) + ": a residual and h go together");
    if (residual && (rc = check_pointers(what, n->dtype, {residual, h})) != CAME8_OK) return rc;
    const RmsArgs a{x, residual, weight, y, h, nullptr, nullptr, n->rows, n->dim, n->ld_x, n->ld_residual, 0, eps_of(n)};
    forward_of<kNormed>(n, a, static_cast<hipStream_t>(stream));
    return op_check_launch("rms_norm_forward");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + e.what());
  }
}

int came8_rms_norm_int8(const came8_rms_norm* n, const void* x, const void* residual, const void* weight, int8_t* q, int64_t ld_q,
                        float* scale, void* h, void* stream) {
  const char* what = "came8_rms_norm_int8";
  try {
    int rc = check(what, n, residual != nullptr);
    if (rc != CAME8_OK || (rc = check_eps(what, n)) != CAME8_OK) return rc;
    if (n->rows == 0) return CAME8_OK;
    if ((rc = check_pointers(what, n->dtype, {x, weight})) != CAME8_OK) return rc;
    if ((rc = check_codes(what, n, q, ld_q, scale)) != CAME8_OK) return rc;
    if ((residual == nullptr) != (h == nullptr)) return op_fail(CAME8_EINVAL, std::string(what) + ": a residual and h go together");
    if (residual && (rc = check_pointers(what, n->dtype, {residual, h})) != CAME8_OK) return rc;
    const RmsArgs a{x, residual, weight, nullptr, h, q, scale, n->rows, n->dim, n->ld_x, n->ld_residual, ld_q, eps_of(n)};
    forward_of<kNormed8>(n, a, static_cast<hipStream_t>(stream));
    return op_check_launch("rms_norm_int8");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + e.what());
  }
}

int came8_quantize_rows(const came8_rms_norm* n, const void* x, int8_t* q, int64_t ld_q, float* scale, void* stream) {
  const char* what = "came8_quantize_rows";
  try {
    int rc = check(what, n, false);
    if (rc != CAME8_OK) return rc;
    if (n->rows == 0) return CAME8_OK;
    if ((rc = check_pointers(what, n->dtype, {x})) != CAME8_OK) return rc;
    if ((rc = check_codes(what, n, q, ld_q, scale)) != CAME8_OK) return rc;
    const RmsArgs a{x, nullptr, nullptr, nullptr, nullptr, q, scale, n->rows, n->dim, n->ld_x, 0, ld_q, 0.0f};
    forward_of<kRows8>(n, a, static_cast<hipStream_t>(stream));
    return op_check_launch("quantize_rows");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + e.what());
  }
}

int came8_rms_norm_workspace_size(const came8_rms_norm* n, size_t* bytes) {
  const char* what = "came8_rms_norm_workspace_size";
  try {
    const int rc = check(what, n, false);
    if (rc != CAME8_OK) return rc;
    if (bytes == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": bytes is NULL");
    *bytes = size_t(std::max<int64_t>(256, 4 * (parts_of(n) * n->dim + (is_long(n) ? n->rows : 0))));
    return CAME8_OK;
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + e.what());
  }
}

int came8_rms_norm_backward(const came8_rms_norm* n, const void* h, const void* weight, const void* dy, const void* dh, void* dx,
                            void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "came8_rms_norm_backward";
  try {
    int rc = check(what, n, false);
    if (rc != CAME8_OK || (rc = check_eps(what, n)) != CAME8_OK) return rc;
    if (n->rows == 0) return op_fail(CAME8_EINVAL, std::string(what) + ": no rows");
    if ((rc = check_pointers(what, n->dtype, {h, weight, dy})) != CAME8_OK) return rc;
    for (const void* p : {dh, static_cast<const void*>(dx), static_cast<const void*>(dweight)})
      if (p != nullptr && (rc = check_pointers(what, n->dtype, {p})) != CAME8_OK) return rc;
    if (dx == nullptr && dweight == nullptr) return CAME8_OK;
    size_t need = 0;
    if ((rc = came8_rms_norm_workspace_size(n, &need)) != CAME8_OK) return rc;
    if (dweight && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < need))
      return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
    const RmsBackArgs a{h, weight, dy, dh, dx, nullptr, n->rows, n->dim, n->ld_x, eps_of(n)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n->dtype == CAME8_F32) backward<F32>(n, a, dweight, workspace, s);
    else if (n->dtype == CAME8_BF16) backward<BF16>(n, a, dweight, workspace, s);
    else backward<F16>(n, a, dweight, workspace, s);
    return op_check_launch("rms_norm_backward");
  } catch (const std::exception& e) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + e.what());
  }
}

}  // extern "C"
