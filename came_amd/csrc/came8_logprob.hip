// Log probabilities of given tokens with entropy and top alternatives, and their gradient.
//
//   m = max z,  s = sum e^(z - m),  t = sum e^(z - m) (z - m),  l = log s
//   log_prob = z[token] - m - l,  entropy = l - t / s,  dz = dlog_prob ([v = token] - p) - dentropy p (log p + entropy)
//
// A row of logits, or a part of it, lies in a workgroup's registers from its one read on.  Bound by memory.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
#include <type_traits>

#include "../../include/came8.h"
#include "came8_ops.h"
#include "came8_rows.h"

namespace came8 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -200.0f;  // e^kFar is 0; in the place of log p where p is 0, so that their product is 0 there too

struct LogProbArgs {
  const void* z;
  const void* tokens;
  float* log_prob;
  float* entropy;
  float* stats;      // [rows][2]: m, l
  float* top_log_prob;
  int64_t* top_token;
  float* part;       // parts > 1: [rows][parts][4]: m, s, t
  uint64_t* keys;    // parts > 1: [rows][parts][top]
  int64_t rows, V, ld;
  int32_t parts, length;  // elements of a part, a multiple of a chunk's
  int32_t top, wide;
};

// A logit and its token as one number: ordered as the values are, of equal ones the lower token the larger; NaN is the largest.
// 0 and the largest number are no logits.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  const uint32_t b = __float_as_uint(x != x ? __uint_as_float(0x7ffffffeu) : x + 0.0f);  // -0 is 0
  return uint64_t(b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u)) << 32 | uint32_t(~token);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = uint32_t(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ int64_t token_of(uint64_t key) { return int64_t(~uint32_t(key)); }

// The `top` largest keys of a workgroup's elements in order, to out(rank, key); key 0 where there are fewer.  best: the thread's
// largest, of numbers.  larger(bound, g) calls g with every key of the thread that is not below the bound (numbers alone), every(g)
// with all of them.
//
// The largest keys of 64 groups of threads bound the top-th key from below: the top-th largest of them.  Of normal logits few keys
// are not below it (23 of 32000 for the top 20, 61 for 40, but more than 300 for 64, whose bound is the least of all groups');
// they go to a list, and each one's place is the number of larger ones.  Where the list is too short, or a NaN is among the
// elements, the largest below the last is looked for `top` times.  That is so for sorted logits, for parts whose logits are all
// equal (a mask's -inf) from the top 17 on, and where fewer than `top` groups have logits: 1 x 32000 in bf16 of which 9 in 10
// are -inf takes 47 us for the top 20 and 125 for 64, without a mask 12 and 22.
constexpr int kList = 1024, kGroups = 64;
struct TopShared {
  uint64_t group[kGroups];
  uint64_t list[kList];
  uint64_t bound;
  int32_t count;
};
template <int CTRL>
__device__ __forceinline__ uint64_t max_dpp(uint64_t v) {
  return max(v, uint64_t(dpp_u32<CTRL>(uint32_t(v >> 32))) << 32 | dpp_u32<CTRL>(uint32_t(v)));
}
template <int TPB, typename F, typename G, typename O>
__device__ __forceinline__ void top_keys(uint64_t best, bool numbers, F&& larger, G&& every, int top, TopShared& s, O&& out) {
  constexpr int kGroup = TPB / kGroups;
  static_assert(kGroup == 1 || kGroup == 8, "");
  const int t = int(threadIdx.x);
  if constexpr (kGroup == 8) best = max_dpp<kDppHalfMirror>(max_dpp<kDppXor2>(max_dpp<kDppXor1>(best)));
  if (t % kGroup == 0) s.group[t / kGroup] = best;
  if (t == 0) {
    s.bound = 1;
    s.count = numbers ? 0 : kList + 1;
  }
  __syncthreads();
  if (t < kGroups) {
    const uint64_t k = s.group[t];
    int above = 0;
#pragma unroll 16
    for (int g = 0; g < kGroups; ++g) above += s.group[g] > k ? 1 : 0;
    if (above == top - 1 && k != 0) s.bound = k;  // keys other than 0 are different
  }
  __syncthreads();
  const uint64_t bound = s.bound;
  if (best >= bound && numbers)
    larger(bound, [&](uint64_t k) {
      const int at = atomicAdd(&s.count, 1);
      if (at < kList) s.list[at] = k;
    });
  __syncthreads();
  const int n = s.count;
  if (n <= kList) {
    for (int i = t; i < n; i += TPB) {
      const uint64_t k = s.list[i];
      int above = 0;
      for (int j = 0; j < n; j += 8) {
#pragma unroll
        for (int u = 0; u < 8; ++u) above += s.list[j + u] > k && j + u < n ? 1 : 0;
      }
      if (above < top) out(above, k);
    }
    for (int r = n + t; r < top; r += TPB) out(r, uint64_t(0));
    return;
  }
  uint64_t last = ~uint64_t(0);
#pragma unroll 1
  for (int r = 0; r < top; ++r) {
    uint64_t k = 0;
    every([&](uint64_t v) { k = v < last ? max(k, v) : k; });
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) k = max_xor(k, o);
    __syncthreads();  // the last round's are read
    if (t % kWave == 0) s.list[t / kWave] = k;
    __syncthreads();
    for (int w = 0; w < TPB / kWave; ++w) k = max(k, s.list[w]);
    if (t == 0) out(r, k);
    last = k;
  }
}

// -inf in every element of a word
template <typename T>
constexpr uint32_t kNone = std::is_same<T, F32>::value ? 0xff800000u : std::is_same<T, BF16>::value ? 0xff80ff80u : 0xfc00fc00u;

// The largest of a thread's elements; fp16: two at a time.  (Where one is a NaN it may be that.)
template <typename T>
struct Maximum {
  float m = -__builtin_inff();
  __device__ __forceinline__ void add(const u32x4& w) {
    float x[kChunk<T>];
    unpack<T>(w, x);
#pragma unroll
    for (int e = 0; e < kChunk<T>; ++e) m = fmaxf(m, x[e]);
  }
  __device__ __forceinline__ float value() const { return m; }
};
template <>
struct Maximum<F16> {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x2 m = {_Float16(-__builtin_inff()), _Float16(-__builtin_inff())};
  __device__ __forceinline__ void add(const u32x4& w) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(f16x2, uint32_t(w[e])));
  }
  __device__ __forceinline__ float value() const { return fmaxf(float(m.x), float(m.y)); }
};

// A part of a row a workgroup of TPB threads, NV chunks a thread.
//
// Rows that have logits of -inf are gone over again with their terms of t bounded, which would cost all rows an instruction a
// logit.  8192 rows of 32000 in bf16: 95 us, 5.5 TB/s.
template <typename T, int TPB, int NV, bool TOP>
__global__ __launch_bounds__(TPB, TPB == kWave ? 1 : 6) void k_logprob(const LogProbArgs a) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>, kStep = TPB * V;
  constexpr int kWaves = TPB / kWave;
  __shared__ float lds[2][5 * kWaves];
  __shared__ typename std::conditional<TOP, TopShared, char>::type shared;
  const int t = int(threadIdx.x);
  const int part = int(blockIdx.y), first = part * a.length, n = int(min(int64_t(a.length), a.V - first));
  int turn = 0;
  // From the last row on, which may still be in the memory-side cache, and the backward pass from the first on, with loads and
  // stores that leave what this pass has read there: 8192 rows of 32000 in bf16 267 us in all; 306 without those hints, 316 with
  // the rows in one order.
  for (int64_t row = a.rows - 1 - blockIdx.x; row >= 0; row -= gridDim.x, turn ^= 1) {
    const S* z = static_cast<const S*>(a.z) + row * a.ld;
    u32x4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const S* at = z + first + i * kStep;
      if ((i + 1) * kStep <= n) raw[i] = *(const CAME8_GLOBAL u32x4b*)(gbl(at) + t * V);  // all threads'
      else raw[i] = load_raw<T>(at, t * V, n - i * kStep, kNone<T>);
    }
    int64_t token = -1;
    float given = 0.0f;
    if (a.parts == 1 && t == 0) {
      token = token_at(a.tokens, row, a.wide);
      if (token >= 0 && token < a.V) given = T::load(gbl(z)[token]);
      else token = -1;
    }
    float own = -__builtin_inff();
    int which = 0;  // TOP: its first place among the thread's elements
    if constexpr (TOP) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[V];
        unpack<T>(raw[i], x);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          which = x[e] > own ? i * V + e : which;
          own = x[e] > own ? x[e] : own;
        }
      }
    } else {
      Maximum<T> largest;
#pragma unroll
      for (int i = 0; i < NV; ++i) largest.add(raw[i]);
      own = largest.value();
    }
    float m = own;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) m = fmaxf(m, __shfl_xor(m, o, kWave));
    if constexpr (kWaves > 1) {
      float* most = lds[turn] + 4 * kWaves;
      if (t % kWave == 0) most[t / kWave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, most[w]);
    }
    const float base = m == -__builtin_inff() ? 0.0f : m;  // a part of -inf alone: s = 0
    float s[2] = {0.0f, 0.0f};  // sums of e^(z - m) and of e^(z - m) (z - m)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[V];
      unpack_again(raw[i]);
      unpack<T>(raw[i], x);
      if ((i + 1) * kStep <= n) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = x[e] - base, p = __builtin_amdgcn_exp2f(d * kLog2e);
          s[0] += p;
          s[1] = fmaf(p, d, s[1]);
        }
      } else {  // past the row's end d is -inf
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = x[e] - base, p = __builtin_amdgcn_exp2f(d * kLog2e);
          s[0] += p;
          s[1] = fmaf(p, fmaxf(d, kFar), s[1]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // a chunk at a time: with all 64 values on their way registers are out
    }
    row_sum<TPB>(s, lds[turn]);
    if (s[1] != s[1]) {  // logits of -inf, whose term is no number
      s[0] = s[1] = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[V];
        unpack_again(raw[i]);
        unpack<T>(raw[i], x);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = x[e] - base, p = __builtin_amdgcn_exp2f(d * kLog2e);
          s[0] += p;
          s[1] = fmaf(p, fmaxf(d, kFar), s[1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      row_sum<TPB>(s, lds[turn] + 2 * kWaves);
    }
    const float l = logf(s[0]);
    if (t == 0) {
      if (a.parts == 1) {
        gbl(a.log_prob)[row] = token >= 0 ? (given - m) - l : 0.0f;
        gbl(a.entropy)[row] = l - s[1] / s[0];
        gbl(a.stats)[2 * row] = m;
        gbl(a.stats)[2 * row + 1] = l;
      } else {
        CAME8_GLOBAL float* p = gbl(a.part) + (row * a.parts + part) * 4;
        p[0] = m;
        p[1] = s[0];
        p[2] = s[1];
      }
    }
    if constexpr (TOP) {
      // chunk i's values and first token, hidden from the compiler: it would keep all of them in registers
      auto values = [&](int i, float(&x)[V]) {
        unpack_again(raw[i]);
        unpack<T>(raw[i], x);
        int at = i * kStep + t * V;
        asm volatile("" : "+v"(at));
        return at;
      };
      const int place = which / V * kStep + t * V + which % V;
      const uint64_t best = place < n ? key_of(own, uint32_t(first + place)) : 0;
      auto larger = [&](uint64_t bound, auto&& g) {
        const float least = value_of(bound);  // a bound of 1 is NaN: then nothing is below it
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float x[V];
          const int at = values(i, x);
          bool any = false;
#pragma unroll
          for (int e = 0; e < V; ++e) any |= !(x[e] < least);
          if (any) {
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (!(x[e] < least) && at + e < n) {
                const uint64_t k = key_of(x[e], uint32_t(first + at + e));
                if (k >= bound) g(k);
              }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto every = [&](auto&& g) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float x[V];
          const int at = values(i, x);
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (at + e < n) g(key_of(x[e], uint32_t(first + at + e)));
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // s is NaN where an element is, and where one is infinite
      top_keys<TPB>(best, s[0] == s[0], larger, every, a.top, shared, [&](int r, uint64_t k) {
        if (a.parts == 1) {
          gbl(a.top_log_prob)[row * a.top + r] = (value_of(k) - m) - l;
          gbl(a.top_token)[row * a.top + r] = token_of(k);
        } else {
          gbl(a.keys)[(row * a.parts + part) * a.top + r] = k;
        }
      });
      __syncthreads();  // before the next row's keys
    }
  }
}

// The parts of a row joined by a workgroup: a lane a part for the sums, and the parts' keys, each in order, merged two lists
// at a time by a wavefront: of two lists the largest 64 are max(one's i-th, the other's 63 - i-th), which a merging network
// puts in order.
constexpr int kMaxTop = 64;
static_assert(kMaxTop == kWave, "a lane a key");
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprob_join(const LogProbArgs a) {
  extern __shared__ uint64_t keys[];  // [parts up to a power of two][64], zeros past a list's end
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave, waves = kThreads / kWave;
  const float none = -__builtin_inff();
  int lists = 1;
  while (lists < a.parts) lists *= 2;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t token = token_at(a.tokens, row, a.wide);
    const bool in = token >= 0 && token < a.V;
    const float z = in ? T::load(gbl(static_cast<const typename T::storage*>(a.z))[row * a.ld + token]) : 0.0f;
    if (a.top > 0) {
      for (int p = wave; p < lists; p += waves)
        keys[p * kWave + lane] = p < a.parts && lane < a.top ? gbl(a.keys)[(row * a.parts + p) * a.top + lane] : 0;
    }
    float m = none, s = 0.0f, t = 0.0f;
    if (lane < a.parts) {
      const CAME8_GLOBAL float* p = gbl(a.part) + (row * a.parts + lane) * 4;
      m = p[0];
      s = p[1];
      t = p[2];
    }
    float most = m;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) most = fmaxf(most, __shfl_xor(most, o, kWave));
    const float d = m - most;  // 0 where both are infinite: then s is NaN
    const float f = m == none ? 0.0f : m == most ? 1.0f : __builtin_amdgcn_exp2f(d * kLog2e);
    const float shifted = f > 0.0f && m != most ? fmaf(s, d, t) : t;
    const float all = wave_sum(f > 0.0f ? s * f : (s == s ? 0.0f : s)), ent = wave_sum(f > 0.0f ? shifted * f : 0.0f);
    const float l = logf(all);
    if (threadIdx.x == 0) {
      gbl(a.log_prob)[row] = in ? (z - most) - l : 0.0f;
      gbl(a.entropy)[row] = l - ent / all;
      gbl(a.stats)[2 * row] = most;
      gbl(a.stats)[2 * row + 1] = l;
    }
    if (a.top == 0) continue;
    for (int left = lists / 2; left > 0; left /= 2) {
      __syncthreads();
      for (int p = wave; p < left; p += waves) {  // lists p and p + left
        uint64_t k = max(keys[p * kWave + lane], keys[(p + left) * kWave + kWave - 1 - lane]);
#pragma unroll
        for (int o = kWave / 2; o > 0; o /= 2) {
          const uint64_t other = uint64_t(uint32_t(__shfl_xor(int(k >> 32), o, kWave))) << 32 | uint32_t(__shfl_xor(int(uint32_t(k)), o, kWave));
          k = (lane & o) == 0 ? max(k, other) : min(k, other);
        }
        keys[p * kWave + lane] = k;
      }
    }
    if (wave == 0 && lane < a.top) {
      const uint64_t k = keys[lane];  // this wavefront's own merge was the last
      gbl(a.top_log_prob)[row * a.top + lane] = (value_of(k) - most) - l;
      gbl(a.top_token)[row * a.top + lane] = token_of(k);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------- gradient
struct LogProbBackArgs {
  const void* z;
  const void* tokens;
  const float* stats;
  const float* entropy;
  const float* dlog_prob;  // or null
  const float* dentropy;   // or null
  void* dz;
  int64_t rows, V, ld;
  int32_t wide;
};

constexpr int kBackChunks = 4;  // a thread
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprob_back(const LogProbBackArgs a) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>;
  const int64_t first = int64_t(blockIdx.y) * (kThreads * kBackChunks * V) + int64_t(threadIdx.x) * V;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t token = token_at(a.tokens, row, a.wide);
    const bool in = token >= 0 && token < a.V;
    const float g = a.dlog_prob && in ? gbl(a.dlog_prob)[row] : 0.0f, gh = a.dentropy ? gbl(a.dentropy)[row] : 0.0f;
    S* to = static_cast<S*>(a.dz) + row * a.V;
    if (g == 0.0f && gh == 0.0f) {
#pragma unroll
      for (int i = 0; i < kBackChunks; ++i) store_raw<T, true>(to, first + i * kThreads * V, a.V, u32x4{0u, 0u, 0u, 0u});
      continue;
    }
    const S* z = static_cast<const S*>(a.z) + row * a.ld;
    u32x4 raw[kBackChunks];
#pragma unroll
    for (int i = 0; i < kBackChunks; ++i) raw[i] = load_raw<T, true>(z, first + i * kThreads * V, a.V);
    const float m = gbl(a.stats)[2 * row], l = gbl(a.stats)[2 * row + 1], h = gbl(a.entropy)[row];
#pragma unroll
    for (int i = 0; i < kBackChunks; ++i) {
      const int64_t e0 = first + i * kThreads * V;
      float x[V];
      unpack<T>(raw[i], x);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float lp = (x[e] - m) - l, p = __builtin_amdgcn_exp2f(lp * kLog2e);
        x[e] = -p * fmaf(gh, fmaxf(lp, kFar) + h, g);
      }
      if (in && token >= e0 && token < e0 + V) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] += e0 + e == token ? g : 0.0f;
      }
      store_chunk<T, true>(to, e0, a.V, x);
    }
  }
}

// ------------------------------------------------------------------------------------------------------ launches
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kMaxGroups = 1 << 20;
constexpr int kPartThreads = 512, kPartChunks = 8;
constexpr int64_t kMaxParts = kWave;                  // a lane each of the join
constexpr int64_t kMaxVocab = int64_t(1) << 20;       // kMaxParts parts of 16384 float32 logits
constexpr int64_t kEnough = 512;                      // workgroups that keep the GPU busy

// How a row is cut: as few parts as registers hold, or as many as keep the GPU busy where there are few rows, of two chunks a thread
// at least (the top 20 of 64 rows of 32000 in bf16 11.2 us, with one chunk 17.7, with four 13.9: every part has lists to join; of
// one row 10.2, 10.3 and 13.0).
struct Cut {
  int64_t parts, length;
};
Cut cut_of(const came8_log_probs* p) {
  const int64_t V = p->dtype == CAME8_F32 ? 4 : 8, chunks = ceil_div(p->vocab, V);
  if (chunks <= kWave * kPartChunks && p->rows >= kEnough) return {1, chunks * V};
  const int64_t least = ceil_div(chunks, kPartThreads * kPartChunks), most = ceil_div(chunks, 2 * kPartThreads);
  int64_t parts = std::min<int64_t>(kMaxParts, std::max(least, std::min(most, kEnough / std::max<int64_t>(1, p->rows))));
  const int64_t each = ceil_div(chunks, parts);
  return {ceil_div(chunks, each), each * V};
}

template <typename T, bool TOP>
void forward(const LogProbArgs& a, hipStream_t stream) {
  const int64_t chunks = a.length / kChunk<T>;
  auto go = [&](auto kernel, int threads) {
    const dim3 grid(unsigned(std::min(a.rows, kMaxGroups / a.parts)), unsigned(a.parts));
    hipLaunchKernelGGL(kernel, grid, dim3(unsigned(threads)), 0, stream, a);
  };
  if (chunks <= kWave * 2) go(k_logprob<T, kWave, 2, TOP>, kWave);
  else if (chunks <= kWave * 8 && a.rows * a.parts >= kEnough) go(k_logprob<T, kWave, 8, TOP>, kWave);
  else if (chunks <= kPartThreads) go(k_logprob<T, kPartThreads, 1, TOP>, kPartThreads);
  else if (chunks <= kPartThreads * 2) go(k_logprob<T, kPartThreads, 2, TOP>, kPartThreads);
  else if (chunks <= kPartThreads * 4) go(k_logprob<T, kPartThreads, 4, TOP>, kPartThreads);
  else go(k_logprob<T, kPartThreads, kPartChunks, TOP>, kPartThreads);
  unsigned lists = 1;
  while (lists < unsigned(a.parts)) lists *= 2;
  if (a.parts > 1)
    hipLaunchKernelGGL(k_logprob_join<T>, dim3(unsigned(std::min(a.rows, kMaxGroups))), dim3(kThreads), a.top > 0 ? lists * kMaxTop * 8 : 0u, stream, a);
}

struct Layout {
  size_t part = 0, keys = 0, bytes = 0;
};
Layout layout_of(const came8_log_probs* p) {
  Layout l;
  const Cut c = cut_of(p);
  if (c.parts == 1) return l;
  l.keys = size_t(p->rows * c.parts) * 16;
  l.bytes = l.keys + size_t(p->rows * c.parts * p->top) * 8;
  return l;
}

int check(const char* what, const came8_log_probs* p) {
  const std::string at = std::string(what) + ": ";
  if (p == nullptr) return op_fail(CAME8_EINVAL, at + "no description given");
  if (p->dtype != CAME8_F32 && p->dtype != CAME8_BF16 && p->dtype != CAME8_F16)
    return op_fail(CAME8_EINVAL, at + "unknown dtype " + std::to_string(p->dtype));
  if (p->token_bytes != 4 && p->token_bytes != 8) return op_fail(CAME8_EINVAL, at + "token_bytes must be 4 or 8");
  if (p->rows < 0 || p->rows >= (int64_t(1) << 31) || p->vocab < 1 || p->vocab > kMaxVocab)
    return op_fail(CAME8_EINVAL, at + "rows must be in [0, 2^31), vocab in [1, 2^20]");
  if (p->ld < p->vocab || p->ld > (int64_t(1) << 31))
    return op_fail(CAME8_EINVAL, at + "a row stride must be at least the row's length and at most 2^31");
  if (p->top < 0 || p->top > 64 || p->top > p->vocab) return op_fail(CAME8_EINVAL, at + "top must be in [0, 64] and at most vocab");
  return CAME8_OK;
}

int check_pointer(const char* what, const void* p, uintptr_t size) {
  if (p != nullptr && reinterpret_cast<uintptr_t>(p) % size == 0) return CAME8_OK;
  return op_fail(CAME8_EINVAL, std::string(what) + ": a null pointer, or one that is not aligned to its type");
}
uintptr_t size_of(int32_t dtype) { return dtype == CAME8_F32 ? 4 : 2; }

template <typename F>
void by_type(int32_t dtype, F&& f) {
  if (dtype == CAME8_F32) f(F32{});
  else if (dtype == CAME8_BF16) f(BF16{});
  else f(F16{});
}

}  // namespace
}  // namespace came8

using namespace came8;

extern "C" {

int came8_log_probs_workspace_size(const came8_log_probs* p, size_t* bytes) {
  const char* what = "came8_log_probs_workspace_size";
  try {
    const int rc = check(what, p);
    if (rc != CAME8_OK) return rc;
    if (bytes == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": bytes is NULL");
    *bytes = layout_of(p).bytes;
    return CAME8_OK;
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

int came8_log_probs_forward(const came8_log_probs* p, const void* logits, const void* tokens, float* log_prob, float* entropy,
                            float* stats, float* top_log_prob, int64_t* top_token, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const char* what = "came8_log_probs_forward";
  try {
    int rc = check(what, p);
    if (rc != CAME8_OK) return rc;
    if (p->rows == 0) return CAME8_OK;
    if ((rc = check_pointer(what, logits, size_of(p->dtype))) != CAME8_OK) return rc;
    if ((rc = check_pointer(what, tokens, uintptr_t(p->token_bytes))) != CAME8_OK) return rc;
    for (const float* q : {log_prob, entropy, stats})
      if ((rc = check_pointer(what, q, 4)) != CAME8_OK) return rc;
    if (p->top > 0 && ((rc = check_pointer(what, top_log_prob, 4)) != CAME8_OK || (rc = check_pointer(what, top_token, 8)) != CAME8_OK))
      return rc;
    const Cut c = cut_of(p);
    const Layout l = layout_of(p);
    if (c.parts > 1 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < l.bytes))
      return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
    char* ws = static_cast<char*>(workspace);
    const LogProbArgs a{logits, tokens, log_prob, entropy, stats, top_log_prob, top_token, reinterpret_cast<float*>(ws),
                        c.parts > 1 ? reinterpret_cast<uint64_t*>(ws + l.keys) : nullptr, p->rows, p->vocab, p->ld, int32_t(c.parts),
                        int32_t(c.length), p->top, p->token_bytes == 8};
    by_type(p->dtype, [&](auto t) {
      if (p->top > 0) forward<decltype(t), true>(a, static_cast<hipStream_t>(stream));
      else forward<decltype(t), false>(a, static_cast<hipStream_t>(stream));
    });
    return op_check_launch("log_probs_forward");
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

int came8_log_probs_backward(const came8_log_probs* p, const void* logits, const void* tokens, const float* stats,
                             const float* entropy, const float* dlog_prob, const float* dentropy, void* dlogits, void* stream) {
  const char* what = "came8_log_probs_backward";
  try {
    int rc = check(what, p);
    if (rc != CAME8_OK) return rc;
    if (p->rows == 0) return CAME8_OK;
    for (const void* q : {logits, static_cast<const void*>(dlogits)})
      if ((rc = check_pointer(what, q, size_of(p->dtype))) != CAME8_OK) return rc;
    if ((rc = check_pointer(what, tokens, uintptr_t(p->token_bytes))) != CAME8_OK) return rc;
    for (const float* q : {stats, entropy})
      if ((rc = check_pointer(what, q, 4)) != CAME8_OK) return rc;
    for (const float* q : {dlog_prob, dentropy})
      if (q != nullptr && (rc = check_pointer(what, q, 4)) != CAME8_OK) return rc;
    if (dlog_prob == nullptr && dentropy == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": no gradient given");
    by_type(p->dtype, [&](auto t) {
      using T = decltype(t);
      const int64_t parts = ceil_div(p->vocab, kThreads * kBackChunks * kChunk<T>);
      const LogProbBackArgs a{logits, tokens, stats, entropy, dlog_prob, dentropy, dlogits, p->rows, p->vocab, p->ld,
                              p->token_bytes == 8};
      hipLaunchKernelGGL(k_logprob_back<T>, dim3(unsigned(std::min(p->rows, kMaxGroups)), unsigned(parts)), dim3(kThreads), 0,
                         static_cast<hipStream_t>(stream), a);
    });
    return op_check_launch("log_probs_backward");
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

}  // extern "C"
