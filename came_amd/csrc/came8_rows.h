// Rows in 16-byte chunks: loads and stores at any address the type allows, and reductions over the threads of a row.  For the
// operators whose work is one pass over rows (norms, 8-bit rows, embeddings, log probabilities).
#pragma once

#include "came8_device.h"

namespace came8 {

// 16 bytes at any address
typedef uint32_t u32x4b __attribute__((ext_vector_type(4), aligned(1)));

// a streamed operand's (came8_device.h: ld_nt, whose template would forget the alignment)
__device__ __forceinline__ u32x4 ld_nt16(const CAME8_GLOBAL u32x4b* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ void st_nt16(CAME8_GLOBAL u32x4b* p, u32x4 v) { __builtin_nontemporal_store(v, p); }

// 8-bit codes
struct I8 {
  using storage = int8_t;
};

// elements of a 16-byte chunk
template <typename T>
constexpr int kChunk = 16 / int(sizeof(typename T::storage));

// Chunk at element e0 of a row of D, zeros past its end, or what `fill` holds in each word.  Rows of odd widths start anywhere: gfx950 loads 16 bytes from any
// address in one instruction.
// NT: a streamed operand, that no one reads again soon.
template <typename T, bool NT = false, typename I>
__device__ __forceinline__ u32x4 load_raw(const typename T::storage* row, I e0, I D, uint32_t fill = 0u) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>;
  const CAME8_GLOBAL S* p = gbl(row) + e0;
  u32x4 w = {fill, fill, fill, fill};
  if (e0 + V <= D) {
    if constexpr (NT) w = ld_nt16((const CAME8_GLOBAL u32x4b*)p);
    else w = *(const CAME8_GLOBAL u32x4b*)p;
  } else if (e0 < D) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e0 + v < D) {
        if constexpr (sizeof(S) == 4) w[v] = __builtin_bit_cast(uint32_t, p[v]);
        else if constexpr (sizeof(S) == 1) w[v / 4] = (w[v / 4] & ~(0xffu << (8 * (v & 3)))) | uint32_t(uint8_t(p[v])) << (8 * (v & 3));
        else w[v / 2] = (v & 1) ? (w[v / 2] & 0xffffu) | uint32_t(p[v]) << 16 : (w[v / 2] & 0xffff0000u) | uint32_t(p[v]);
      }
  }
  return w;
}

// Nothing is known of w from here on: what was unpacked of it before is not kept in registers beside it.
__device__ __forceinline__ void unpack_again(u32x4& w) { asm volatile("" : "+v"(w)); }

template <typename T>
__device__ __forceinline__ void unpack(const u32x4& raw, float (&x)[kChunk<T>]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int v = 0; v < kChunk<T>; ++v) x[v] = T::elem(w, v);
}

template <typename T, typename I>
__device__ __forceinline__ void load_chunk(const typename T::storage* row, I e0, I D, float (&x)[kChunk<T>]) {
  unpack<T>(load_raw<T>(row, e0, D), x);
}

template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&x)[kChunk<T>]) {
  u32x4 w;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    if constexpr (kChunk<T> == 4) w[v] = __float_as_uint(x[v]);
    else w[v] = uint32_t(T::store(x[2 * v])) | uint32_t(T::store(x[2 * v + 1])) << 16;
  }
  return w;
}

template <typename T, bool NT = false, typename I>
__device__ __forceinline__ void store_raw(typename T::storage* row, I e0, I D, const u32x4& w) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>;
  CAME8_GLOBAL S* p = gbl(row) + e0;
  if (e0 + V <= D) {
    if constexpr (NT) st_nt16((CAME8_GLOBAL u32x4b*)p, w);
    else *(CAME8_GLOBAL u32x4b*)p = w;
  } else if (e0 < D) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e0 + v < D) {
        if constexpr (sizeof(S) == 4) p[v] = __builtin_bit_cast(S, uint32_t(w[v]));
        else p[v] = S(w[v / 2] >> (16 * (v & 1)));
      }
  }
}

template <typename T, bool NT = false, typename I>
__device__ __forceinline__ void store_chunk(typename T::storage* row, I e0, I D, const float (&x)[kChunk<T>]) {
  store_raw<T, NT>(row, e0, D, pack<T>(x));
}

// Sums over groups of L lanes, L = 16 or 64, in a fixed order
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(L == 16 || L == 64, "");
  v += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(v)));
  if constexpr (L == 64) {
    v += __uint_as_float(swz_xor16_u32(__float_as_uint(v)));
    v = __uint_as_float(readlane_u32(__float_as_uint(v), 0)) + __uint_as_float(readlane_u32(__float_as_uint(v), 32));
  }
  return v;
}

// N sums at once over the TPR threads of a row (a group of 16 lanes, a wavefront, or all of the workgroup).  lds: N * TPR / 64
// floats, not in use by the one before (callers alternate between two).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = lanes_sum<TPR < kWave ? TPR : kWave>(v[n]);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) lds[n * W + threadIdx.x / kWave] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = lds[n * W];
#pragma unroll
      for (int w = 1; w < W; ++w) v[n] += lds[n * W + w];
    }
  }
}

// the largest of unsigned words over the TPR threads of a row; lds: TPR / 64 words
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* lds) {
  v = group_max_bits<TPR < kWave ? TPR : kWave>(v);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v = max(v, lds[w]);
  }
  return v;
}

__device__ __forceinline__ uint64_t max_xor(uint64_t v, int o) {
  const uint64_t w = uint64_t(uint32_t(__shfl_xor(int(v >> 32), o, kWave))) << 32 | uint32_t(__shfl_xor(int(uint32_t(v)), o, kWave));
  return max(v, w);
}

// the same of 64 bits; lds: 2 * TPR / 64 words, 8 bytes aligned
template <int TPR>
__device__ __forceinline__ uint64_t row_max64(uint64_t v, uint32_t* lds) {
#pragma unroll
  for (int o = 1; o < (TPR < kWave ? TPR : kWave); o *= 2) v = max_xor(v, o);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    uint64_t* all = reinterpret_cast<uint64_t*>(lds);
    if (threadIdx.x % kWave == 0) all[threadIdx.x / kWave] = v;
    __syncthreads();
    v = all[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v = max(v, all[w]);
  }
  return v;
}

// token i of a list of 4- or 8-byte ones
__device__ __forceinline__ int64_t token_at(const void* tokens, int64_t i, bool wide) {
  return wide ? gbl(static_cast<const int64_t*>(tokens))[i] : int64_t(gbl(static_cast<const int32_t*>(tokens))[i]);
}

}  // namespace came8
