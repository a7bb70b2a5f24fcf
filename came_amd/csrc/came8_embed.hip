// The embedding of tokens, y[i] = scale * weight[token[i]], and its gradient: the positions sorted by their tokens in one launch,
// the rows of dy summed over even shares of the sorted positions, and the shares of the tokens that several have joined.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>

#include "../../include/came8.h"
#include "came8_ops.h"
#include "came8_rows.h"
#include "came8_shares.h"

namespace came8 {
namespace {

struct EmbedArgs {
  const void* tokens;
  const void* w;
  void* y;
  int64_t T, V, D, ld;
  float scale;
  int32_t wide;  // tokens of 8 bytes
};

// TPR threads a row.  Bound by memory, and for few tokens by the launch.
template <typename T, int TPR>
__global__ __launch_bounds__(kThreads) void k_embed(const EmbedArgs a) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>, kRows = kThreads / TPR;
  for (int64_t i = int64_t(blockIdx.x) * kRows + int(threadIdx.x) / TPR; i < a.T; i += int64_t(gridDim.x) * kRows) {
    const int64_t token = token_at(a.tokens, i, a.wide);
    const bool in = token >= 0 && token < a.V;
    const S* from = static_cast<const S*>(a.w) + (in ? token : 0) * a.ld;
    S* to = static_cast<S*>(a.y) + i * a.D;
    const int64_t end = in ? a.D : 0;
#pragma unroll 2
    for (int64_t e = int64_t(int(threadIdx.x) % TPR) * V; e < a.D; e += TPR * V) {
      const u32x4 raw = load_raw<T>(from, e, end);
      if (a.scale == 1.0f) {
        store_raw<T>(to, e, a.D, raw);
      } else {
        float x[V];
        unpack<T>(raw, x);
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = in ? x[v] * a.scale : 0.0f;
        store_chunk<T>(to, e, a.D, x);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------- gradient
struct EmbedBackArgs {
  const void* tokens;
  const void* dy;
  void* dw;
  int32_t* count;    // of sorted positions
  int32_t* position; // [T], sorted by their tokens, and by themselves
  int32_t* token;    // [T], theirs
  int32_t* cross;    // [shares]: of the token at a share's last position, if it begins there and goes on, the last share that has it;
                     // else -1
  uint64_t* empty;   // [ceil(V / range)][kSortWaves]: a workgroup's tokens that have no position
  float* part;       // [shares][2][D]
  int64_t T, V, D, padding;
  int32_t range;     // tokens a workgroup of the sort
  int32_t share;     // sorted positions a workgroup of the sum
  float scale;
  int32_t wide;
};

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortUnroll = 8;     // tokens a lane has in flight; 8192 in all are read once
constexpr int kMaxRange = 1000;    // tokens a workgroup: a thread each, and its counters fit 64 KiB

// Every workgroup has `range` tokens and looks through all positions for them: twice, first to count (its own, by wavefront and
// token, and those below its range, which tell where its part of the sorted list begins), then to place.  A wavefront takes a
// run of successive positions and places them 64 at a time, so that the order is that of the positions; the lanes that have the
// same token find each other by ballots on its bits (the first range has half of a text's tokens: one token at a time, its
// workgroup took 34 us for 8192 positions, 10 so).  No workgroup waits for another.  The tokens stay in L2.
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const EmbedBackArgs a) {
  extern __shared__ int32_t counts[];  // [kSortWaves][range], then kSortWaves + 1 words
  int32_t* extra = counts + kSortWaves * a.range;
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
  const int64_t first = int64_t(blockIdx.x) * a.range;
  const int64_t last = min(first + a.range, a.V);
  const int64_t run = ((a.T + kSortWaves - 1) / kSortWaves + kWave - 1) / kWave * kWave;
  const int64_t from = min(run * wave, a.T), to = min(from + run, a.T);
  for (int k = int(threadIdx.x); k < kSortWaves * a.range; k += kSortThreads) counts[k] = 0;
  __syncthreads();
  int32_t* mine = counts + wave * a.range;
  int32_t below = 0;
  auto look = [&](int64_t i) {  // the token at i, -1 where it has no gradient
    const int64_t t = i < to ? token_at(a.tokens, i, a.wide) : -1;
    return t < a.V && t != a.padding ? t : -1;
  };
  int32_t key[kSortUnroll];  // of the tokens in flight, less the first of the range; -1 for one of another range
  auto fetch = [&](int64_t i, bool count) __attribute__((always_inline)) {
    int64_t t[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) t[u] = look(i + u * kWave + lane);
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      key[u] = t[u] >= first && t[u] < last ? int32_t(t[u] - first) : -1;
      if (count) below += t[u] >= 0 && t[u] < first ? 1 : 0;
    }
  };
  for (int64_t i = from; i < to; i += kWave * kSortUnroll) {
    fetch(i, true);
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u)
      if (key[u] >= 0) atomicAdd(&mine[key[u]], 1);
  }
  below = wave_sum(below);
  if (lane == 0) extra[wave] = below;
  __syncthreads();
  // thread r: token first + r; where each wavefront's positions of it go
  const int r = int(threadIdx.x);
  int32_t all = 0, start = 0;
  if (r < a.range)
    for (int w = 0; w < kSortWaves; ++w) all += counts[w * a.range + r];
  int32_t scan = all;  // of the wavefront's tokens up to this one
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const int32_t v = __shfl_up(scan, o, kWave);
    scan += lane >= o ? v : 0;
  }
  for (int w = 0; w < kSortWaves; ++w) start += extra[w];
  __syncthreads();
  if (lane == kWave - 1) extra[wave] = scan;
  __syncthreads();
  for (int w = 0; w < wave; ++w) start += extra[w];
  start += scan - all;
  if (r < a.range) {
    int32_t at = start;
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t n = counts[w * a.range + r];
      counts[w * a.range + r] = at;
      at += n;
    }
  }
  if (blockIdx.x + 1 == gridDim.x && r == kSortThreads - 1) gbl(a.count)[0] = start + all;
  __syncthreads();
  const int bits = 32 - __builtin_clz(a.range);
  for (int64_t i = from; i < to; i += kWave * kSortUnroll) {
    if (run > kWave * kSortUnroll) fetch(i, false);  // else they are there
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const bool here = key[u] >= 0;
      uint64_t same = __builtin_amdgcn_ballot_w64(here);  // the lanes with this one's token
      if (same == 0) continue;
      for (int b = 0; b < bits; ++b) {
        const bool one = key[u] >> b & 1;
        const uint64_t ones = __builtin_amdgcn_ballot_w64(one);
        same &= one ? ones : ~ones;
      }
      const int before = __builtin_popcountll(same & ((uint64_t(1) << lane) - 1));
      int32_t at = 0;
      if (here && before == 0) at = atomicAdd(&mine[key[u]], __builtin_popcountll(same));
      at = __shfl(at, __builtin_ctzll(same | uint64_t(1) << 63), kWave) + before;
      if (here) {
        gbl(a.position)[at] = int32_t(i + u * kWave + lane);
        gbl(a.token)[at] = int32_t(first + key[u]);
      }
    }
  }
  const uint64_t empty = __builtin_amdgcn_ballot_w64(r < a.range && first + r < last && all == 0);
  if (lane == 0) gbl(a.empty)[int64_t(blockIdx.x) * kSortWaves + wave] = empty;
  // the shares that end within this token's positions
  share_ends(start, all, a.share, [&](int64_t s, int32_t last) { gbl(a.cross)[s] = last; });
}

// The rows of dy of `share` successive sorted positions, TPR threads by their 16-byte chunks, summed by token.  A token whose
// positions end here and began here is written; of one that goes on or began before, the sum goes to part[share][0] (began
// before) or part[share][1] (begins here and goes on).  Workgroups past the shares' clear the rows without a token
// meanwhile, with stores that leave the caches to the others (8192 of 32000 x 4096 in bf16, all of the call: 111 us without, 93).
constexpr int kAhead = 8;      // rows in flight
constexpr int kClear = 16;     // tokens a workgroup that clears, of one word of `empty`
template <typename T>
__global__ __launch_bounds__(kThreads) void k_embed_sum(const EmbedBackArgs a, const int shares) {
  using S = typename T::storage;
  constexpr int V = kChunk<T>;
  if (int(blockIdx.x) >= shares) {
    if (blockIdx.y > 0) return;
    const int64_t id = int64_t(blockIdx.x) - shares, words = (a.range + kWave - 1) / kWave, word = id / (kWave / kClear);
    const int bit = int(id % (kWave / kClear)) * kClear;
    const int64_t group = word / words, of = word - group * words;
    const int64_t v0 = group * a.range + of * kWave + bit;
    uint64_t empty = gbl(a.empty)[group * kSortWaves + of] >> bit & ((uint64_t(1) << kClear) - 1);
    while (empty != 0) {
      S* row = static_cast<S*>(a.dw) + (v0 + __builtin_ctzll(empty)) * a.D;
      empty &= empty - 1;
      for (int64_t e = int64_t(threadIdx.x) * V; e < a.D; e += kThreads * V) store_raw<T, true>(row, e, a.D, u32x4{0u, 0u, 0u, 0u});
    }
    return;
  }
  const int32_t n = gbl(a.count)[0];
  const int64_t begin = int64_t(blockIdx.x) * a.share, end = min(begin + a.share, int64_t(n));
  if (begin >= end) return;
  const int64_t e0 = (int64_t(blockIdx.y) * kThreads + threadIdx.x) * V;
  const int lane = int(threadIdx.x) % kWave;
  const int32_t before = begin > 0 ? gbl(a.token)[begin - 1] : -1;  // (a sorted token is never -1)
  float sum[V] = {};
  for (int64_t base = begin; base < end; base += kWave) {
    // a lane has the position and token of one of 64 successive ones, and the token after
    const int64_t mine = base + lane;
    const int32_t position = mine < end ? gbl(a.position)[mine] : 0, token = mine < end ? gbl(a.token)[mine] : -1;
    const int32_t after = mine < end && mine + 1 < n ? gbl(a.token)[mine + 1] : -1;
    const int count = int(min(end - base, int64_t(kWave)));
    auto row = [&](int k) {
      return load_raw<T>(static_cast<const S*>(a.dy) + int64_t(__builtin_amdgcn_readlane(position, k)) * a.D, e0, a.D);
    };
    u32x4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (u < count) raw[u] = row(u);
    for (int k0 = 0; k0 < count; k0 += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u;
        if (k >= count) break;
        float x[V];
        unpack<T>(raw[u], x);
        if (k + kAhead < count) raw[u] = row(k + kAhead);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += x[v];
        const int32_t of = __builtin_amdgcn_readlane(token, k), next = __builtin_amdgcn_readlane(after, k);
        const bool goes_on = next == of;
        if (goes_on && base + k + 1 < end) continue;
        const bool began = of == before;
        if (!goes_on && !began) {
#pragma unroll
          for (int v = 0; v < V; ++v) sum[v] *= a.scale;
          store_chunk<T>(static_cast<S*>(a.dw) + int64_t(of) * a.D, e0, a.D, sum);
        } else {
          float* part = a.part + (int64_t(blockIdx.x) * 2 + (began ? 0 : 1)) * a.D;
#pragma unroll
          for (int v = 0; v < V; v += 4) store_chunk<F32>(part, e0 + v, a.D, {sum[v], sum[v + 1], sum[v + 2], sum[v + 3]});
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] = 0.0f;
      }
    }
  }
}

// The tokens that begin in a share and go on: their sums from there on, 256 columns a workgroup, a quarter of the shares a
// wavefront.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_embed_join(const EmbedBackArgs a) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ float lds[kWaves][kWave * 4];
  const int64_t first = blockIdx.x, end = (first + 1) * a.share;
  if (end >= gbl(a.count)[0]) return;
  const int32_t last = gbl(a.cross)[first];
  if (last < 0) return;
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
  const int64_t c = int64_t(blockIdx.y) * (kWave * 4) + lane * 4;
  const int64_t shares = last - first + 1, each = (shares + kWaves - 1) / kWaves;
  const int64_t from = min(each * wave, shares), to = min(from + each, shares);
  float sum[4] = {};
#pragma unroll 8
  for (int64_t k = from; k < to; ++k) {
    float x[4];
    load_chunk<F32>(a.part + ((first + k) * 2 + (k == 0 ? 1 : 0)) * a.D, c, a.D, x);
#pragma unroll
    for (int v = 0; v < 4; ++v) sum[v] += x[v];
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) lds[wave][lane * 4 + v] = sum[v];
  __syncthreads();
  const int64_t col = int64_t(blockIdx.y) * (kWave * 4) + int(threadIdx.x);
  if (col < a.D) {
    float s = lds[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s += lds[w][threadIdx.x];
    gbl(static_cast<typename T::storage*>(a.dw))[int64_t(gbl(a.token)[end]) * a.D + col] = T::store(s * a.scale);
  }
}

// ------------------------------------------------------------------------------------------------------ launches
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up(int64_t n, int64_t a) { return ceil_div(n, a) * a; }

constexpr int64_t kMaxGroups = 1 << 20;

template <typename T>
void forward(const EmbedArgs& a, hipStream_t stream) {
  constexpr int V = kChunk<T>;
  auto go = [&](auto kernel, int64_t rows) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(std::min(ceil_div(a.T, rows), kMaxGroups))), dim3(kThreads), 0, stream, a);
  };
  if (a.D <= 16 * V) go(k_embed<T, 16>, 16);
  else if (a.D <= 64 * V) go(k_embed<T, 64>, 4);
  else go(k_embed<T, 256>, 1);
}

// Sorted positions a share: enough shares for all of the GPU where there are few positions, and at most 2048 of them, whose
// sums are 2 rows in float32 each.
int64_t share_of(const came8_embedding* e) { return std::max<int64_t>(16, ceil_div(e->tokens, 2048)); }
int64_t shares_of(const came8_embedding* e) { return ceil_div(e->tokens, share_of(e)); }
// tokens a workgroup of the sort: 256 workgroups, one on each CU, unless its counters are too many
int64_t range_of(const came8_embedding* e) { return std::min<int64_t>(kMaxRange, std::max<int64_t>(16, ceil_div(e->vocab, 256))); }

struct Layout {
  size_t count = 0, position = 0, token = 0, cross = 0, empty = 0, part = 0, bytes = 0;
};
Layout layout_of(const came8_embedding* e) {
  Layout l;
  l.position = 256;
  l.token = l.position + size_t(up(e->tokens * 4, 256));
  l.cross = l.token + size_t(up(e->tokens * 4, 256));
  l.empty = l.cross + size_t(up(shares_of(e) * 4, 256));
  l.part = l.empty + size_t(up(ceil_div(e->vocab, range_of(e)) * kSortWaves * 8, 256));
  l.bytes = l.part + size_t(shares_of(e) * 2 * e->dim * 4);
  return l;
}

template <typename T>
void backward(const came8_embedding* e, const EmbedBackArgs& a, hipStream_t stream) {
  const int64_t groups = ceil_div(e->vocab, a.range), clear = groups * ceil_div(a.range, kWave) * (kWave / kClear);
  hipLaunchKernelGGL(k_embed_sort, dim3(unsigned(groups)), dim3(kSortThreads), unsigned((kSortWaves * a.range + kSortWaves + 1) * 4), stream, a);
  const int shares = int(shares_of(e));
  hipLaunchKernelGGL(k_embed_sum<T>, dim3(unsigned(shares + clear), unsigned(ceil_div(e->dim, kThreads * kChunk<T>))), dim3(kThreads), 0,
                     stream, a, shares);
  if (shares > 1)
    hipLaunchKernelGGL(k_embed_join<T>, dim3(unsigned(shares - 1), unsigned(ceil_div(e->dim, kWave * 4))), dim3(kThreads), 0, stream, a);
}

int check(const char* what, const came8_embedding* e) {
  const std::string at = std::string(what) + ": ";
  if (e == nullptr) return op_fail(CAME8_EINVAL, at + "no description given");
  if (e->dtype != CAME8_F32 && e->dtype != CAME8_BF16 && e->dtype != CAME8_F16)
    return op_fail(CAME8_EINVAL, at + "unknown dtype " + std::to_string(e->dtype));
  if (e->token_bytes != 4 && e->token_bytes != 8) return op_fail(CAME8_EINVAL, at + "token_bytes must be 4 or 8");
  const int64_t most = int64_t(1) << 31;
  if (e->tokens < 0 || e->tokens >= most || e->vocab < 1 || e->vocab > (int64_t(1) << 26) || e->dim < 1 || e->dim > (int64_t(1) << 23))
    return op_fail(CAME8_EINVAL, at + "tokens must be in [0, 2^31), vocab in [1, 2^26], dim in [1, 2^23]");
  if (e->ld_weight < e->dim || e->ld_weight > most)
    return op_fail(CAME8_EINVAL, at + "a row stride must be at least the row's length and at most 2^31");
  if (e->padding < -1 || e->padding >= e->vocab) return op_fail(CAME8_EINVAL, at + "padding must be a token or -1");
  return CAME8_OK;
}

// every pointer is there and aligned to its elements of `size` bytes
int check_pointer(const char* what, const void* p, uintptr_t size) {
  if (p != nullptr && reinterpret_cast<uintptr_t>(p) % size == 0) return CAME8_OK;
  return op_fail(CAME8_EINVAL, std::string(what) + ": a null pointer, or one that is not aligned to its type");
}
uintptr_t size_of(int32_t dtype) { return dtype == CAME8_F32 ? 4 : 2; }

}  // namespace
}  // namespace came8

using namespace came8;

extern "C" {

int came8_embedding_forward(const came8_embedding* e, const void* tokens, const void* weight, void* y, void* stream) {
  const char* what = "came8_embedding_forward";
  try {
    int rc = check(what, e);
    if (rc != CAME8_OK) return rc;
    if (e->tokens == 0) return CAME8_OK;
    if ((rc = check_pointer(what, tokens, uintptr_t(e->token_bytes))) != CAME8_OK) return rc;
    for (const void* p : {weight, static_cast<const void*>(y)})
      if ((rc = check_pointer(what, p, size_of(e->dtype))) != CAME8_OK) return rc;
    const EmbedArgs a{tokens, weight, y, e->tokens, e->vocab, e->dim, e->ld_weight, e->scale, e->token_bytes == 8};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (e->dtype == CAME8_F32) forward<F32>(a, s);
    else if (e->dtype == CAME8_BF16) forward<BF16>(a, s);
    else forward<F16>(a, s);
    return op_check_launch("embedding_forward");
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

int came8_embedding_workspace_size(const came8_embedding* e, size_t* bytes) {
  const char* what = "came8_embedding_workspace_size";
  try {
    const int rc = check(what, e);
    if (rc != CAME8_OK) return rc;
    if (bytes == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": bytes is NULL");
    *bytes = layout_of(e).bytes;
    return CAME8_OK;
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

int came8_embedding_backward(const came8_embedding* e, const void* tokens, const void* dy, void* dweight, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* what = "came8_embedding_backward";
  try {
    int rc = check(what, e);
    if (rc != CAME8_OK) return rc;
    if (e->tokens == 0) return op_fail(CAME8_EINVAL, std::string(what) + ": no tokens");
    if ((rc = check_pointer(what, tokens, uintptr_t(e->token_bytes))) != CAME8_OK) return rc;
    for (const void* p : {dy, static_cast<const void*>(dweight)})
      if ((rc = check_pointer(what, p, size_of(e->dtype))) != CAME8_OK) return rc;
    const Layout l = layout_of(e);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < l.bytes)
      return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
    char* ws = static_cast<char*>(workspace);
    const EmbedBackArgs a{tokens, dy, dweight, reinterpret_cast<int32_t*>(ws), reinterpret_cast<int32_t*>(ws + l.position),
                          reinterpret_cast<int32_t*>(ws + l.token), reinterpret_cast<int32_t*>(ws + l.cross),
                          reinterpret_cast<uint64_t*>(ws + l.empty), reinterpret_cast<float*>(ws + l.part), e->tokens, e->vocab, e->dim,
                          e->padding, int32_t(range_of(e)), int32_t(share_of(e)), e->scale, e->token_bytes == 8};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (e->dtype == CAME8_F32) backward<F32>(e, a, s);
    else if (e->dtype == CAME8_BF16) backward<BF16>(e, a, s);
    else backward<F16>(e, a, s);
    return op_check_launch("embedding_backward");
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

}  // extern "C"
