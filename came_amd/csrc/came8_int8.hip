// The product of 8-bit rows, y[i][j] = (sum over k of q[i][k] w[j][k]) * scale[i] * w_scale[j] + bias[j]: the sums exact in 32 bits
// by v_mfma_i32_16x16x64_i8, the rest in the epilogue.
//
// A few rows read the weights once and are bound by that; more go through tiles in LDS.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>

#include "../../include/came8.h"
#include "came8_ffn.h"
#include "came8_ops.h"
#include "came8_rows.h"

namespace came8 {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

struct Int8Args {
  const int8_t* q;
  const float* scale;
  const int8_t* w;
  const float* w_scale;
  const void* bias;  // or null
  void* y;
  int32_t* part;     // splits > 1: the shares of the sums, [splits][M][N up to a multiple of 4]
  int64_t ld_q, ld_w;
  int32_t M, N, K;
  int32_t tiles_m, tiles_n, splits;
};

// What four successive columns from n on of row m are scaled by, and their bias
struct Scales {
  float s, w[4], b[4];
};
template <typename T>
__device__ __forceinline__ Scales scales_of(const Int8Args& a, int64_t m, int n) {
  Scales o{gbl(a.scale)[m], {}, {}};
  load4(a.w_scale, n, a.N, o.w);
  if (a.bias != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o.b[e] = n + e < a.N ? T::load(gbl(static_cast<const typename T::storage*>(a.bias))[n + e]) : 0.0f;
  }
  return o;
}
// y of them
template <typename T>
__device__ __forceinline__ void store_scaled(const Int8Args& a, int64_t m, int n, const i32x4& c, const Scales& o) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = float(c[e]) * o.s * o.w[e] + o.b[e];
  store4<T>(static_cast<typename T::storage*>(a.y) + m * a.N, n, a.N, y);
}
template <typename T>
__device__ __forceinline__ void store_scaled(const Int8Args& a, int64_t m, int n, const i32x4& c) {
  store_scaled<T>(a, m, n, c, scales_of<T>(a, m, n));
}

// -------------------------------------------------------------------------------------------------- few rows
// 16 codes from e0 on of a row of K, at least 16, zeros past its end: the row's last 16, shifted, where K cuts them
__device__ __forceinline__ u32x4 load_cut(const int8_t* row, int e0, int K) {
  const int left = K - e0, over = left <= 0 ? 16 : left < 16 ? 16 - left : 0;
  u32x4 v = *(const CAME8_GLOBAL u32x4b*)gbl(row + (left < 16 ? K - 16 : e0));
  const int words = over / 4;
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t far = e + 3 < 4 ? v[3] : 0u, two = e + 2 < 4 ? v[e + 2 < 4 ? e + 2 : 3] : 0u, one = e + 1 < 4 ? v[e + 1 < 4 ? e + 1 : 3] : 0u;
    w[e] = words == 0 ? v[e] : words == 1 ? one : words == 2 ? two : words == 3 ? far : 0u;
  }
  u32x4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = __builtin_amdgcn_alignbyte(e < 3 ? w[e < 3 ? e + 1 : 3] : 0u, w[e], over & 3);
  return out;
}

// One or two rows of q: a wavefront reads rows of weights whole, 1024 codes in a load, four rows and 4096 codes at a time, and
// takes four products in an instruction (v_dot4_i32_i8); q's codes stay in registers.  Matrix instructions want 64 codes of 16 rows
// in a load, which memory gives more slowly (1 x 4096 x 32000 21 us, 6.2 TB/s, instead of 28).
template <typename T, int M>
__global__ __launch_bounds__(kThreads) void k_int8_vector(const Int8Args a) {
  constexpr int R = 4, C = 4, kStep = kWave * 16;
  const int lane = int(threadIdx.x) % kWave, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int n0 = (int(blockIdx.x) * (kThreads / kWave) + wave) * R;
  if (n0 >= a.N) return;
  const int8_t* w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) w[r] = a.w + int64_t(min(n0 + r, a.N - 1)) * a.ld_w;
  int32_t acc[R][M] = {};
  for (int k0 = 0; k0 < a.K; k0 += C * kStep) {
    u32x4 wf[R][C], x[M][C];
    auto load = [&](const int8_t* row, int c, bool stream) __attribute__((always_inline)) {
      const int e0 = k0 + c * kStep + lane * 16;
      if (k0 + (c + 1) * kStep <= a.K) {  // all lanes'
        const CAME8_GLOBAL u32x4b* p = (const CAME8_GLOBAL u32x4b*)(gbl(row) + e0);
        return stream ? ld_nt16(p) : u32x4(*p);
      }
      return k0 + c * kStep < a.K ? load_cut(row, e0, a.K) : u32x4{0u, 0u, 0u, 0u};
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) wf[r][c] = load(w[r], c, true);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int c = 0; c < C; ++c) x[m][c] = load(a.q + int64_t(min(m, a.M - 1)) * a.ld_q, c, false);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int m = 0; m < M; ++m) acc[r][m] = __builtin_amdgcn_sdot4(int(wf[r][c][e]), int(x[m][c][e]), acc[r][m], false);
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
    i32x4 sum;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint32_t v = uint32_t(acc[r][m]);
      v += dpp_u32<kDppXor1>(v);
      v += dpp_u32<kDppXor2>(v);
      v += dpp_u32<kDppHalfMirror>(v);
      v += dpp_u32<kDppMirror>(v);
      v += swz_xor16_u32(v);
      sum[r] = int32_t(readlane_u32(v, 0) + readlane_u32(v, 32));
    }
    if (lane == m && m < a.M) store_scaled<T>(a, m, n0, sum);
  }
}

// 16 rows of weights at a time for a workgroup, an eighth of k a wavefront: fragments go from memory to the matrix instructions,
// and the wavefronts' sums are joined in LDS.  FM: 16 rows of q each.
//
// DEEP steps of 64 codes are loaded together.  AHEAD (16 rows of q at most): the weights' next ones meanwhile, those of the
// workgroup's next 16 rows too; two workgroups on a CU.  Without, a workgroup has 16 rows alone, and its loads are as deep as
// registers go: where there are no more than 256 of them, what counts is how often a wavefront waits.
template <typename T, int FM, int DEEP, bool AHEAD>
__global__ __launch_bounds__(512, AHEAD ? 4 : 2) void k_int8_few(const Int8Args a) {
  constexpr int kWaves = 8;
  static_assert(FM * 64 <= 512, "a thread a store");
  __shared__ i32x4 lds[AHEAD ? 2 : 1][kWaves][FM * 64];
  const int lane = int(threadIdx.x) % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);  // k's bounds are scalar so
  const int steps = a.K / 64, first = steps * wave / kWaves, last = steps * (wave + 1) / kWaves;  // what is left: the last wavefront's
  const int blocks = (a.N + 15) / 16;
  const int8_t* x[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f) x[f] = a.q + int64_t(min(f * 16 + r, a.M - 1)) * a.ld_q;  // rows past M are not stored
  auto row = [&](int b) { return a.w + int64_t(min(b * 16 + r, a.N - 1)) * a.ld_w; };
  u32x4 wf[AHEAD ? 2 : 1][DEEP], xf[DEEP][FM];
  // steps from s on of block b's weights; none past the last of either
  auto fetch_w = [&](u32x4(&to)[DEEP], int b, int s) __attribute__((always_inline)) {
    const CAME8_GLOBAL int8_t* w = gbl(row(b)) + g * 16;
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      to[d] = u32x4{0u, 0u, 0u, 0u};
      if (s + d < last && b < blocks) to[d] = *(const CAME8_GLOBAL u32x4b*)(w + (s + d) * 64);
    }
  };
  auto fetch_x = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int f = 0; f < FM; ++f) {
        xf[d][f] = u32x4{0u, 0u, 0u, 0u};
        if (s + d < last) xf[d][f] = *(const CAME8_GLOBAL u32x4b*)(gbl(x[f]) + g * 16 + (s + d) * 64);
      }
  };
  const bool once = FM == 1 && last - first <= DEEP;  // q's fragments stay in registers
  int turn = 0;
  fetch_w(wf[0], blockIdx.x, first);
  if (once) fetch_x(first);
  for (int b = blockIdx.x; b < blocks; b += AHEAD ? int(gridDim.x) : blocks, turn ^= 1) {
    i32x4 acc[FM] = {};
    const int m = int(threadIdx.x) / 4, n = b * 16 + int(threadIdx.x) % 4 * 4;  // of the result's that the thread stores
    const bool stores = int(threadIdx.x) < FM * 64 && m < a.M && n < a.N;
    const bool cut = wave == kWaves - 1 && a.K % 64 != 0;
    u32x4 wc, xc[FM];
    auto fetch_cut = [&]() __attribute__((always_inline)) {
      wc = load_cut(row(b), steps * 64 + g * 16, a.K);
#pragma unroll
      for (int f = 0; f < FM; ++f) xc[f] = load_cut(x[f], steps * 64 + g * 16, a.K);
    };
    // With the other loads, where registers hold them (48 x 5461 x 2048 14.4 us in all; where they are used 15.6)
    Scales scales;
    if constexpr (!AHEAD) {
      if (stores) scales = scales_of<T>(a, m, n);
      if (cut) fetch_cut();
    }
    for (int s = first;; s += DEEP) {
      const bool more = s + DEEP < last;
      if (!once) fetch_x(s);
      if constexpr (AHEAD) fetch_w(wf[1], more ? b : b + int(gridDim.x), more ? s + DEEP : first);
#pragma unroll
      for (int d = 0; d < DEEP; ++d)
#pragma unroll
        for (int f = 0; f < FM; ++f) acc[f] = mfma_i8(wf[0][d], xf[d][f], acc[f]);
      if constexpr (AHEAD) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) wf[0][d] = wf[1][d];
      } else if (more) {
        fetch_w(wf[0], b, s + DEEP);
      }
      if (!more) break;
    }
    if (cut) {
      if (AHEAD) fetch_cut();
#pragma unroll
      for (int f = 0; f < FM; ++f) acc[f] = mfma_i8(wc, xc[f], acc[f]);
    }
    // a lane holds columns 4 g to 4 g + 3 of row r
    i32x4(&part)[kWaves][FM * 64] = lds[AHEAD ? turn : 0];
#pragma unroll
    for (int f = 0; f < FM; ++f) part[wave][f * 64 + r * 4 + g] = acc[f];
    __syncthreads();  // what is read below is written again after the next block's
    if (stores) {
      i32x4 c = part[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) c += part[k][threadIdx.x];
      if constexpr (AHEAD) store_scaled<T>(a, m, n, c);
      else store_scaled<T>(a, m, n, c, scales);
    }
  }
}

// ------------------------------------------------------------------------------------------------------ tiles
// Tiles of B by B on 2 by WAVES_N wavefronts.  A step is 128 codes of k; its four phases are laid out as in the feed-forward
// block's products (came8_ffn.h), and so are the rows in LDS.
//
// Codes of normal values, inputs in turn: 8192 x 4096 x 11008 374 to 415 us (1970 to 1780 TOP/s; the library's unscaled product 405
// beside the 415), 8192 x 11008 x 4096 325 to 340, 2048 x 4096 x 4096 42 to 45, 128 x 4096 x 11008 23 to 25.  By the counters, a
// step of a large tile takes 3330 cycles, of which matrix instructions have 2048 and LDS 1280 (no conflicts; a CU reads 234 bytes
// a cycle in this layout): neither is the limit, and what a step waits for beside them is not known.  A tile's first loads and its
// epilogue take 31 thousand cycles that nothing overlaps, as much as 9 steps: 8192 x 4096 x 11008 is 5.4 rounds of tiles of 32
// steps, paid as 6.  What was slower: operands loaded straight to LDS in steps of 64 codes, four or five in flight (438, 346, 48,
// 22); four wavefronts of 128 by 128 (459); the weights' fragments loaded from memory past LDS (517 where this took 394).
template <typename T, int B, int WAVES_N>
__global__ __launch_bounds__(2 * WAVES_N * kWave, 2) void k_int8_gemm(const Int8Args args) {
  constexpr int NT = 2 * WAVES_N * kWave, BK = kRowBytes, kTileBytes = 2 * B * kRowBytes;
  constexpr int WM = B / 2, WN = B / WAVES_N, FM = WM / 16, FN = WN / 16;
  __shared__ __attribute__((aligned(16))) char lds[2 * kTileBytes];

  int tm, tn, split;
  {
    const int b = int(blockIdx.x), tiles = args.tiles_m * args.tiles_n, all = tiles * args.splits;
    const int each = all / kXcds, more = all % kXcds, x = b % kXcds;
    int id = x * each + min(x, more) + b / kXcds;
    split = id / tiles;
    id -= split * tiles;
    constexpr int kGroup = 8;
    const int first = id / (kGroup * args.tiles_n) * kGroup, rows = min(kGroup, args.tiles_m - first);
    const int in = id - first * args.tiles_n;
    tm = first + in % rows;
    tn = in / rows;
  }
  const int m0 = tm * B, n0 = tn * B;
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
  const int wm = wave % 2, wn = wave / 2;

  constexpr int D = B < 256 ? 2 : 1;
  Stage<I8, B, NT, true> sa[D], sb[D];
  const int steps = (args.K + BK - 1) / BK;
  const int begin = int(int64_t(steps) * split / args.splits), total = int(int64_t(steps) * (split + 1) / args.splits) - begin;
  auto view = [&](const int8_t* p, int64_t ld, int at, int extent) {
    View v;
    v.p = reinterpret_cast<const char*>(p) + at * ld;
    v.left = view_bytes(true, extent - at, args.K, ld, 1);
    v.step = kRowBytes;
    v.ld = int32_t(ld);
    v.next(begin);
    return v;
  };
  View va = view(args.q, args.ld_q, m0, args.M), vb = view(args.w, args.ld_w, n0, args.N);
  int left = args.K - begin * BK;
  auto fetch = [&](int slot) __attribute__((always_inline)) {
    sa[slot].fetch(va, va, left);
    sb[slot].fetch(vb, vb, left);
    // a chunk that K cuts: what is past K in q's becomes zero, so w's does not count
    if (__builtin_expect(left > 0 && left < BK && left % 16 != 0, 0)) {
      const int in = left - int(threadIdx.x & 7) * 16;
      if (in > 0 && in < 16) {
#pragma unroll
        for (int i = 0; i < Stage<I8, B, NT, true>::kLoads; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int bytes = in - 4 * e;
            sa[slot].v[i][e] &= bytes >= 4 ? ~0u : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1u;
          }
      }
    }
    va.next();
    vb.next();
    left -= BK;
  };
  i32x4 acc[FM][FN] = {};
  auto put = [&](int t, int slot) __attribute__((always_inline)) {
    char* to = lds + (t & 1) * kTileBytes;
    sa[slot].put(to);
    sb[slot].put(to + B * kRowBytes);
  };
  const int fr = lane % 16;
  uint32_t pa[4], pb[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    pa[v] = uint32_t((wm * WM + fr) * kRowBytes + (lane / 16 ^ swz(wm * (WM % 64) + fr) ^ (2 * v)) * kChunkBytes);
    pb[v] = uint32_t((B + wn * WN + fr) * kRowBytes + (lane / 16 ^ swz(wn * (WN % 64) + fr) ^ (2 * v)) * kChunkBytes);
  }
  u32x4 lo[FM / 2], hi[FM / 2], fb[2][FN];
  auto read_a = [&](u32x4(&f)[FM / 2], int t, int s, int i0) __attribute__((always_inline)) {
    const char* a = lds + (t & 1) * kTileBytes;
#pragma unroll
    for (int i = 0; i < FM / 2; ++i)
      f[i] = *reinterpret_cast<const u32x4*>(a + pa[(4 * s ^ swz(16 * (i0 + i))) / 2] + (i0 + i) * 16 * kRowBytes);
  };
  auto read_b = [&](int t, int s) __attribute__((always_inline)) {
    const char* b = lds + (t & 1) * kTileBytes;
#pragma unroll
    for (int j = 0; j < FN; ++j)
      fb[s][j] = *reinterpret_cast<const u32x4*>(b + pb[(4 * s ^ swz(16 * j)) / 2] + j * 16 * kRowBytes);
  };
  auto multiply = [&](const u32x4(&f)[FM / 2], int s, int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM / 2; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i0 + i][j] = mfma_i8(fb[s][j], f[i], acc[i0 + i][j]);
  };
  constexpr int kProducts = FM / 2 * FN;  // of a phase
  fetch(0);
  put(0, 0);
#pragma unroll
  for (int d = 1; d <= D; ++d) fetch(d % D);
  __syncthreads();
  read_a(lo, 0, 0, 0);
  read_b(0, 0);
  auto step = [&](int t, int slot) __attribute__((always_inline)) {  // slot: of step t + 1
    read_a(hi, t, 0, FM / 2);
    read_b(t, 1);
    multiply(lo, 0, 0);
    interleave<kDsRead, FM / 2 + FN, kProducts>();
    read_a(lo, t, 1, 0);
    put(t + 1, slot);
    fetch(slot);
    multiply(hi, 0, FM / 2);
    interleave<kDsRead | kDsWrite | kVmemRead, FM / 2 + FM + FN + 8, kProducts>();
    read_a(hi, t, 1, FM / 2);
    multiply(lo, 1, 0);
    interleave<kDsRead, FM / 2, kProducts>();
    __syncthreads();  // every wavefront has read its last of step t, and written its part of step t + 1
    __builtin_amdgcn_sched_barrier(0);
    read_a(lo, t + 1, 0, 0);
    read_b(t + 1, 0);
    multiply(hi, 1, FM / 2);
    interleave<kDsRead, FM / 2 + FN, kProducts>();
  };
  for (int t = 0; t < total; t += D)
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (d == 0 || t + d < total) step(t + d, (d + 1) % D);

  // acc[i][j][e]: row 16 i + lane % 16 of the wavefront's, column 16 j + 4 (lane / 16) + e; through the wavefront's own part of
  // LDS, so that lanes of successive columns write memory together
  constexpr int kPart = FM < 4 ? FM : 4, kChunks = WN / 4;
  constexpr int kRows = kWave / kChunks, kRounds = kPart * 16 / kRows;
  char* mine = lds + wave * (kPart * 16 * WN * 4);
  const int cc = lane % kChunks, r0 = lane / kChunks, n = n0 + wn * WN + cc * 4;
  auto slot = [&](int r, int c) { return reinterpret_cast<i32x4*>(mine + r * (WN * 4) + ((c ^ r) & (kChunks - 1)) * 16); };
  const int pitch = (args.N + 3) & ~3;
  __syncthreads();
#pragma unroll
  for (int part = 0; part < FM / kPart; ++part) {
#pragma unroll
    for (int i = 0; i < kPart; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) *slot(i * 16 + lane % 16, j * 4 + lane / 16) = acc[part * kPart + i][j];
    const int m1 = m0 + wm * WM + part * kPart * 16 + r0;
#pragma unroll 4
    for (int q = 0; q < kRounds; ++q) {
      const int64_t m = m1 + q * kRows;
      if (m >= args.M || n >= args.N) continue;
      const i32x4 c = *slot(q * kRows + r0, cc);
      if (args.part) *(CAME8_GLOBAL i32x4*)gbl(args.part + (int64_t(split) * args.M + m) * pitch + n) = c;
      else store_scaled<T>(args, m, n, c);
    }
  }
}

// y from the shares of split sums
template <typename T>
__global__ __launch_bounds__(kThreads) void k_int8_join(const Int8Args a) {
  const int pitch = (a.N + 3) & ~3;
  const int64_t chunks = int64_t(a.M) * (pitch / 4), share = int64_t(a.M) * pitch;
  for (int64_t id = int64_t(blockIdx.x) * kThreads + threadIdx.x; id < chunks; id += int64_t(gridDim.x) * kThreads) {
    const int64_t m = id / (pitch / 4);
    const int n = int(id - m * (pitch / 4)) * 4;
    const CAME8_GLOBAL int32_t* p = gbl(a.part) + m * pitch + n;
    i32x4 c = *(const CAME8_GLOBAL i32x4*)p;
    for (int s = 1; s < a.splits; ++s) c += *(const CAME8_GLOBAL i32x4*)(p + s * share);
    store_scaled<T>(a, m, n, c);
  }
}

// Rows copied to `ld` bytes apart, a multiple of 16, zeros to there
__global__ __launch_bounds__(kThreads) void k_int8_pack(const int8_t* p, int64_t ld_p, int8_t* to, int64_t ld, int64_t rows, int32_t K) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = int(threadIdx.x) * 16; c < ld; c += kThreads * 16) *(CAME8_GLOBAL u32x4*)gbl(to + r * ld + c) = load_raw<I8>(p + r * ld_p, c, K);
}

// ------------------------------------------------------------------------------------------------------ launches
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up(int64_t n, int64_t a) { return ceil_div(n, a) * a; }

// Up to 16 rows read the weights once; so do up to 64 where there are no more than 256 times 16 rows of weights, which a workgroup
// each reads in one or two batches of loads (48 x 5461 x 2048 16.0 us, in tiles 17.3; 24 x 4096 x 4096 15.6 and 18.9; but 40 x
// 11008 x 4096 28.2 and 23.5, 64 x 4096 x 11008 34.7 and 22.2).  Rows that do not hold 16 codes go through tiles, which copy them.
bool is_few(const came8_int8_linear* l) { return l->in >= 16 && (l->rows <= 16 || (l->rows <= 64 && l->out <= 4096 && l->in <= 6144)); }
constexpr int64_t kAtOnce = 512;                  // workgroups of 512 threads that the GPU holds at once, two on a CU
constexpr int64_t kMaxStride = int64_t(1) << 20;  // bytes: a tile's 256 rows stay below 2^31
constexpr int64_t kMaxIn = 131071;                // 2^31 - 1 holds that many products of -128 by -128

struct Cut {
  int tile = 0, splits = 1;
};
// What a tile size runs at: workgroups at once on the GPU, and a step of k (128 codes) of one, microseconds.
struct Speed {
  int tile, at_once;
  double step;
};
constexpr Speed kSpeeds[] = {{256, 256, 1.87}, {128, 512, 1.22}, {64, 1024, 1.19}};
constexpr int kSplitSteps = 4;  // of 128 codes
constexpr int kMaxSplits = 8;
constexpr double kJoinBytes = 4e6;

// The cut with the least estimated time: rounds of workgroups by their steps, three more for the first loads and the epilogue,
// and what joining the shares moves.
Cut cut_of(const came8_int8_linear* l) {
  Cut best;
  double least = 1e300;
  const int64_t steps = ceil_div(l->in, kRowBytes);
  for (const Speed& v : kSpeeds) {
    const int64_t tiles = ceil_div(l->rows, v.tile) * ceil_div(l->out, v.tile);
    for (int s = 1; s <= kMaxSplits; ++s) {
      if (s > 1 && steps / s < kSplitSteps) break;
      const double t = double(ceil_div(tiles * s, v.at_once)) * (double(ceil_div(steps, s)) + 3.0) * v.step +
                       (s > 1 ? 4.0 + double(s) * double(l->rows) * double(l->out) * 8.0 / kJoinBytes : 0.0);
      if (t < least) {
        least = t;
        best.tile = v.tile;
        best.splits = s;
      }
    }
  }
  return best;
}

struct Layout {
  int64_t ld = 0;  // of the copies of operands whose rows do not all start on words, which tiles load
  bool copy_q = false, copy_w = false;
  size_t q = 0, w = 0, part = 0, bytes = 0;
};
Layout layout_of(const came8_int8_linear* l) {
  Layout o;
  if (!is_few(l)) {
    o.ld = up(l->in, 16);
    o.copy_q = l->ld_q % 4 != 0;
    o.copy_w = l->ld_w % 4 != 0;
    o.w = o.copy_q ? size_t(up(l->rows * o.ld, 256)) : 0;
    o.part = o.w + (o.copy_w ? size_t(up(l->out * o.ld, 256)) : 0);
    const Cut c = cut_of(l);
    o.bytes = o.part + (c.splits > 1 ? size_t(c.splits * l->rows * up(l->out, 4) * 4) : 0);
  }
  return o;
}

template <typename T>
void forward(const came8_int8_linear* l, Int8Args a, char* ws, hipStream_t stream) {
  if (is_few(l)) {
    const int64_t blocks = ceil_div(l->out, 16);
    const dim3 fours{unsigned(blocks)}, each{unsigned(blocks)}, ahead{unsigned(std::min(blocks, kAtOnce))};
    // with fewer rows of weights the wavefronts that read them whole are too few (1 x 11008 x 4096 17.5 us, 16.2 so; 1 x 4096 x 32000
    // 25.0 and 32.0; 4 rows 33.6 and 32.4)
    if (l->rows == 1 && blocks >= kAtOnce) hipLaunchKernelGGL((k_int8_vector<T, 1>), fours, dim3(kThreads), 0, stream, a);
    else if (l->rows == 2 && blocks >= kAtOnce) hipLaunchKernelGGL((k_int8_vector<T, 2>), fours, dim3(kThreads), 0, stream, a);
    else if (l->rows <= 16) hipLaunchKernelGGL((k_int8_few<T, 1, 8, true>), ahead, dim3(512), 0, stream, a);
    else if (l->rows <= 32) hipLaunchKernelGGL((k_int8_few<T, 2, 12, false>), each, dim3(512), 0, stream, a);
    else if (l->rows <= 48) hipLaunchKernelGGL((k_int8_few<T, 3, 11, false>), each, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((k_int8_few<T, 4, 8, false>), each, dim3(512), 0, stream, a);
    return;
  }
  const Layout o = layout_of(l);
  auto copy = [&](const int8_t*& p, int64_t& ld, int64_t rows, size_t at) {
    int8_t* to = reinterpret_cast<int8_t*>(ws + at);
    hipLaunchKernelGGL(k_int8_pack, dim3(unsigned(std::min<int64_t>(rows, 1 << 16))), dim3(kThreads), 0, stream, p, ld, to, o.ld, rows, a.K);
    p = to;
    ld = o.ld;
  };
  if (o.copy_q) copy(a.q, a.ld_q, l->rows, o.q);
  if (o.copy_w) copy(a.w, a.ld_w, l->out, o.w);
  const Cut c = cut_of(l);
  a.tiles_m = int32_t(ceil_div(l->rows, c.tile));
  a.tiles_n = int32_t(ceil_div(l->out, c.tile));
  a.splits = c.splits;
  a.part = c.splits > 1 ? reinterpret_cast<int32_t*>(ws + o.part) : nullptr;
  const dim3 grid(unsigned(a.tiles_m) * unsigned(a.tiles_n) * unsigned(a.splits));
  if (c.tile == 256) hipLaunchKernelGGL((k_int8_gemm<T, 256, 4>), grid, dim3(512), 0, stream, a);
  else if (c.tile == 128) hipLaunchKernelGGL((k_int8_gemm<T, 128, 2>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((k_int8_gemm<T, 64, 2>), grid, dim3(256), 0, stream, a);
  if (a.part)
    hipLaunchKernelGGL(k_int8_join<T>, dim3(unsigned(std::min<int64_t>(ceil_div(l->rows * ceil_div(l->out, 4), kThreads), 1 << 14))),
                       dim3(kThreads), 0, stream, a);
}

int check(const char* what, const came8_int8_linear* l) {
  const std::string at = std::string(what) + ": ";
  if (l == nullptr) return op_fail(CAME8_EINVAL, at + "no description given");
  if (l->dtype != CAME8_F32 && l->dtype != CAME8_BF16 && l->dtype != CAME8_F16)
    return op_fail(CAME8_EINVAL, at + "unknown dtype " + std::to_string(l->dtype));
  if (l->rows < 0 || l->rows > (int64_t(1) << 24) || l->in < 1 || l->in > kMaxIn || l->out < 1 || l->out > (int64_t(1) << 24))
    return op_fail(CAME8_EINVAL, at + "rows must be in [0, 2^24], in in [1, 131071], out in [1, 2^24]");
  for (const int64_t ld : {l->ld_q, l->ld_w})
    if (ld < l->in || ld > kMaxStride)
      return op_fail(CAME8_EINVAL, at + "a row stride must be at least the row's length and at most 2^20");
  if (l->rows * l->out > (int64_t(1) << 36)) return op_fail(CAME8_EINVAL, at + "a result of more than 2^36 elements");
  return CAME8_OK;
}

int check_pointer(const char* what, const void* p, uintptr_t size) {
  if (p != nullptr && reinterpret_cast<uintptr_t>(p) % size == 0) return CAME8_OK;
  return op_fail(CAME8_EINVAL, std::string(what) + ": a null pointer, or one that is not aligned to its type");
}

}  // namespace
}  // namespace came8

using namespace came8;

extern "C" {

int came8_int8_linear_workspace_size(const came8_int8_linear* l, size_t* bytes) {
  const char* what = "came8_int8_linear_workspace_size";
  try {
    const int rc = check(what, l);
    if (rc != CAME8_OK) return rc;
    if (bytes == nullptr) return op_fail(CAME8_EINVAL, std::string(what) + ": bytes is NULL");
    *bytes = layout_of(l).bytes;
    return CAME8_OK;
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

int came8_int8_linear_forward(const came8_int8_linear* l, const int8_t* q, const float* scale, const int8_t* w,
                              const float* w_scale, const void* bias, void* y, void* workspace, size_t workspace_bytes,
                              void* stream) {
  const char* what = "came8_int8_linear_forward";
  try {
    int rc = check(what, l);
    if (rc != CAME8_OK) return rc;
    if (l->rows == 0) return CAME8_OK;
    const uintptr_t size = l->dtype == CAME8_F32 ? 4 : 2;
    if ((rc = check_pointer(what, q, 1)) != CAME8_OK || (rc = check_pointer(what, w, 1)) != CAME8_OK ||
        (rc = check_pointer(what, scale, 4)) != CAME8_OK || (rc = check_pointer(what, w_scale, 4)) != CAME8_OK ||
        (rc = check_pointer(what, y, size)) != CAME8_OK || (bias != nullptr && (rc = check_pointer(what, bias, size)) != CAME8_OK))
      return rc;
    if (!is_few(l))
      for (const auto& [p, ld] : {std::pair(q, l->ld_q), std::pair(w, l->ld_w)})
        if (ld % 4 == 0 && (rc = check_pointer(what, p, 4)) != CAME8_OK) return rc;
    const Layout o = layout_of(l);
    if (o.bytes > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < o.bytes))
      return op_fail(CAME8_ESPACE, std::string(what) + ": workspace too small or misaligned");
    const Int8Args a{q, scale, w, w_scale, bias, y, nullptr, l->ld_q, l->ld_w, int32_t(l->rows), int32_t(l->out), int32_t(l->in), 0, 0, 1};
    hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    if (l->dtype == CAME8_F32) forward<F32>(l, a, ws, s);
    else if (l->dtype == CAME8_BF16) forward<BF16>(l, a, ws, s);
    else forward<F16>(l, a, ws, s);
    return op_check_launch("int8_linear_forward");
  } catch (const std::exception& x) {
    return op_fail(CAME8_EINVAL, std::string(what) + ": " + x.what());
  }
}

}  // extern "C"
