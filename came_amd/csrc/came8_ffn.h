// Matrix-product kernels of the gated feed-forward block for gfx950: C = A B^T over tiles held in registers, with the
// block's elementwise parts in the products' epilogues.
//
// One kernel serves all products of the block and its gradients.  Either operand lies in memory with the summed index
// contiguous ("rows") or with the other one contiguous ("columns"); a thread that loads columns transposes its small
// block in registers on the way to LDS, so no product needs a transposed copy of a weight or an activation.
#pragma once

#include <type_traits>

#include "came8_device.h"

namespace came8 {

// --------------------------------------------------------------------------------------------- element types
// 16 bytes of one row are a chunk; a fragment of v_mfma_f32_16x16x* is one chunk a lane: lane l holds row l % 16 and
// chunk l / 16 of four.  bf16 and fp16: one instruction takes the whole chunk (k = 32).  fp32: four instructions of
// k = 4, the j-th on the j-th element of every lane's chunk; both operands permute k alike.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x4 mfma_chunk(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, BF16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (std::is_same<T, F16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
}

// ----------------------------------------------------------------------------------------------- activations
enum { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

// act(g) and its derivative
__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

__device__ __forceinline__ float act_value(float g, int act) {
  if (act == kSilu) return g * sigmoid(g);
  if (act == kGelu) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
  const float k = 0.79788456080286536f;
  return 0.5f * g * (1.0f + tanhf(k * (g + 0.044715f * g * g * g)));
}

__device__ __forceinline__ float act_slope(float g, int act) {
  if (act == kSilu) {
    const float s = sigmoid(g);
    return s * (1.0f + g * (1.0f - s));
  }
  if (act == kGelu) {
    const float c = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    return c + g * expf(-0.5f * g * g) * 0.39894228040143268f;
  }
  const float k = 0.79788456080286536f;
  const float t = tanhf(k * (g + 0.044715f * g * g * g));
  const float q = 1.0f - t * t;  // 0 long before g * g overflows
  return 0.5f * (1.0f + t) + (q > 0.0f ? 0.5f * g * q * k * (1.0f + 3.0f * 0.044715f * g * g) : 0.0f);
}

// ------------------------------------------------------------------------------------------------- arguments
// One operand: ROWS: element (r, k) at p[r * ld + k]; columns: at p[k * ld + r].
struct Operand {
  const void* p;
  int64_t ld;
};
struct Segment {  // sums over several segments continue in the same accumulators
  Operand a, b;
};
enum Epilogue { kStore, kGate, kBack };

struct GemmArgs {
  Segment seg[2];
  Operand b2;       // kGate: the up projection's weights
  int32_t nseg;
  int32_t M, N, K;  // K: of each segment
  int32_t tiles_m, tiles_n;
  int32_t act;
  void* out;        // kStore: C; kGate: h; kBack: dg
  int64_t ldo;
  void* out2;       // kBack: du
  void* out3;       // kBack: h, or null
  float* g;         // kGate: where to keep g and u (null: not kept); kBack: where they are kept
  float* u;
  int64_t ldg;
};

// A tile's view of an operand: reads past the matrix's end give zeros, whatever the tile.  The hardware checks words, and
// rows start on words (k_ffn_pack), so the last word may count whole: it holds a byte of the matrix.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer view_at(const void* p, int64_t skip, int64_t total) {
  const int64_t left = total - skip;
  const int64_t bytes = left <= 0 ? 0 : ((left + 3) & ~int64_t(3));
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p) + (left <= 0 ? 0 : skip)), 0,
                                           bytes > 0xfffffffcll ? 0xfffffffcu : uint32_t(bytes), 0x00027000);
}

constexpr int kChunkBytes = 16;
constexpr int kRowBytes = 128;  // of a tile in LDS: 8 chunks, 64 (fp32: 32) values of k

// Chunk c of row r lies at place c ^ swz(r) of its row: eight lanes that read one chunk of eight consecutive rows, or write
// one chunk of rows 8 apart (columns on their way in), touch eight different places, which is all banks once.
__device__ __forceinline__ int swz(int r) { return (r ^ (r >> 3)) & 7; }

// ------------------------------------------------------------------------------------------------ operands' way in
// R rows by 8 chunks of k, 256 threads: 16-byte loads into registers (fetch), later written to LDS (put).
template <typename T, int R, bool ROWS>
struct Stage {
  static constexpr int kElem = int(sizeof(typename T::storage));
  static constexpr int kVec = kChunkBytes / kElem;        // elements of a chunk
  static constexpr int kLoads = R / 32;                   // 16-byte loads a thread
  static constexpr int kGroups = kThreads / (R / kVec);   // columns: groups of k values, kLoads each
  u32x4 v[kLoads];

  __device__ __forceinline__ uint32_t offset(int64_t ld) const {
    const int t = int(threadIdx.x);
    if constexpr (ROWS) return uint32_t((t >> 3) * ld * kElem + (t & 7) * kChunkBytes);
    return uint32_t((t / (R / kVec)) * kLoads * ld * kElem + (t % (R / kVec)) * kChunkBytes);
  }
  // rows: rows 32 apart; columns: successive k
  __device__ __forceinline__ void fetch(Buffer a, uint32_t off, int64_t ld) {
    const uint32_t step = uint32_t((ROWS ? 32 : 1) * ld * kElem);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(a, off + i * step, 0, 0);
  }
  // rows split over two buffers by halves of `half` rows (the gate's and the up projection's weights)
  __device__ __forceinline__ void fetch2(Buffer a0, Buffer a1, uint32_t off0, uint32_t off1, int64_t ld0, int64_t ld1, int half) {
    static_assert(ROWS, "");
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = 32 * i, piece = row / half;
      const int src = (piece >> 1) * half + row % half;  // row of its matrix's tile
      v[i] = (piece & 1) ? __builtin_amdgcn_raw_buffer_load_b128(a1, off1 + uint32_t(src * ld1 * kElem), 0, 0)
                         : __builtin_amdgcn_raw_buffer_load_b128(a0, off0 + uint32_t(src * ld0 * kElem), 0, 0);
    }
  }
  // rows: k >= left becomes zero (left counts from the tile's first k)
  __device__ __forceinline__ void mask(int left) {
    if constexpr (ROWS) {
      const int k0 = (int(threadIdx.x) & 7) * kVec;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (kElem == 4) {
            if (k0 + w >= left) v[i][w] = 0;
          } else {
            if (k0 + 2 * w >= left) v[i][w] = 0;
            else if (k0 + 2 * w + 1 >= left) v[i][w] &= 0xffffu;
          }
        }
    }
  }
  __device__ __forceinline__ void put(char* lds) const {
    const int t = int(threadIdx.x);
    if constexpr (ROWS) {
      const int c = t & 7, r = t >> 3;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *reinterpret_cast<u32x4*>(lds + (r + 32 * i) * kRowBytes + ((c ^ swz(r + 32 * i)) * kChunkBytes)) = v[i];
    } else if constexpr (kElem == 4) {
      const int r = (t % (R / kVec)) * kVec, k = (t / (R / kVec)) * kLoads;  // first row, first k
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < kLoads / 4; ++c)
          *reinterpret_cast<u32x4*>(lds + (r + e) * kRowBytes + (((k / 4 + c) ^ swz(r + e)) * kChunkBytes)) =
              u32x4{v[4 * c][e], v[4 * c + 1][e], v[4 * c + 2][e], v[4 * c + 3][e]};
    } else {
      const int r = (t % (R / kVec)) * kVec, k = (t / (R / kVec)) * kLoads;
      // v[j] word w holds columns 2w, 2w + 1 of k + j: halves of two words make one word of a row
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t w[kLoads / 2];
#pragma unroll
        for (int j = 0; j < kLoads / 2; ++j)
          w[j] = __builtin_amdgcn_perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
        char* at = lds + (r + e) * kRowBytes + (((k / 8) ^ swz(r + e)) * kChunkBytes) + (k % 8) * 2;
        if constexpr (kLoads == 8) *reinterpret_cast<u32x4*>(at) = u32x4{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<u32x2*>(at) = u32x2{w[0], w[1]};
      }
    }
  }
};

// ------------------------------------------------------------------------------------------------------ product
// Workgroups of 4 wavefronts, 2 by 2, on a tile of BM by BN.  kGate: the tile's BN rows of weights are, in turns of BN / 4,
// gate and up projection, so that a wavefront holds both values of its BN / 4 columns of h.
template <typename T, int BM, int BN, bool AROWS, bool BROWS, Epilogue EPI>
__global__ __launch_bounds__(kThreads, BM == 256 ? 1 : 2) void k_ffn_gemm(const GemmArgs args) {
  using S = typename T::storage;
  constexpr int kElem = int(sizeof(S));
  constexpr int BK = kRowBytes / kElem;
  constexpr int WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16;
  constexpr int kHalf = BN / 4;
  constexpr int kTileBytes = (BM + BN) * kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[2 * kTileBytes];

  const int tm = int(blockIdx.x) % args.tiles_m, tn = int(blockIdx.x) / args.tiles_m;
  const int m0 = tm * BM, n0 = tn * (EPI == kGate ? BN / 2 : BN);
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
  const int wm = wave & 1, wn = wave >> 1;

  Stage<T, BM, AROWS> sa;
  Stage<T, BN, BROWS> sb;
  const int steps = (args.K + BK - 1) / BK, total = steps * args.nseg;
  auto view = [&](const Operand& o, bool rows, int at, int extent, int k0) {
    const int64_t skip = (rows ? int64_t(at) * o.ld + k0 : int64_t(k0) * o.ld + at) * kElem;
    const int64_t end = (rows ? int64_t(extent - 1) * o.ld + args.K : int64_t(args.K - 1) * o.ld + extent) * kElem;
    return view_at(o.p, skip, end);
  };
  auto fetch = [&](int t) {
    const int s = t >= steps ? 1 : 0, k0 = (t - s * steps) * BK;
    const Segment& seg = args.seg[s];
    sa.fetch(view(seg.a, AROWS, m0, args.M, k0), sa.offset(seg.a.ld), seg.a.ld);
    if constexpr (EPI == kGate)
      sb.fetch2(view(seg.b, true, n0, args.N, k0), view(args.b2, true, n0, args.N, k0), sb.offset(seg.b.ld),
                sb.offset(args.b2.ld), seg.b.ld, args.b2.ld, kHalf);
    else
      sb.fetch(view(seg.b, BROWS, n0, args.N, k0), sb.offset(seg.b.ld), seg.b.ld);
    if (k0 + BK > args.K) {
      sa.mask(args.K - k0);
      sb.mask(args.K - k0);
    }
  };
  auto put = [&](int t) {
    char* to = lds + (t & 1) * kTileBytes;
    sa.put(to);
    sb.put(to + BM * kRowBytes);
  };

  f32x4 acc[FM][FN] = {};
  fetch(0);
  for (int t = 0; t < total; ++t) {
    put(t);
    if (t + 1 < total) fetch(t + 1);
    __syncthreads();
    const char* at = lds + (t & 1) * kTileBytes;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 a[FM], b[FN];
      const int c = s * 4 + lane / 16;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = wm * WM + i * 16 + lane % 16;
        a[i] = *reinterpret_cast<const u32x4*>(at + r * kRowBytes + (c ^ swz(r)) * kChunkBytes);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int r = wn * WN + j * 16 + lane % 16;
        b[j] = *reinterpret_cast<const u32x4*>(at + (BM + r) * kRowBytes + (c ^ swz(r)) * kChunkBytes);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma_chunk<T>(b[j], a[i], acc[i][j]);
    }
  }

  // acc[i][j][e]: row m0 + wm WM + 16 i + lane % 16, column n0 + wn WN + 16 j + 4 (lane / 16) + e (kGate: of the weights' rows)
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm * WM + i * 16 + lane % 16;
    if (m >= args.M) continue;
#pragma unroll
    for (int j = 0; j < (EPI == kGate ? FN / 2 : FN); ++j) {
      const int n = n0 + wn * (EPI == kGate ? kHalf : WN) + j * 16 + (lane / 16) * 4;
      if (n >= args.N) continue;
      const int64_t o = int64_t(m) * args.ldo + n, og = int64_t(m) * args.ldg + n;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= args.N) break;
        if constexpr (EPI == kStore) {
          static_cast<S*>(args.out)[o + e] = T::store(acc[i][j][e]);
        } else if constexpr (EPI == kGate) {
          const float g = acc[i][j][e], u = acc[i][j + FN / 2][e];
          static_cast<S*>(args.out)[o + e] = T::store(act_value(g, args.act) * u);
          if (args.g) {
            args.g[og + e] = g;
            args.u[og + e] = u;
          }
        } else {
          const float g = args.g[og + e], u = args.u[og + e], dh = acc[i][j][e], a = act_value(g, args.act);
          static_cast<S*>(args.out)[o + e] = T::store(dh * u * act_slope(g, args.act));
          static_cast<S*>(args.out2)[o + e] = T::store(dh * a);
          if (args.out3) static_cast<S*>(args.out3)[o + e] = T::store(a * u);
        }
      }
    }
  }
}

// Rows of 16-bit elements at an odd stride, copied to an even one: a row that starts in the middle of a word would have its
// last element in a word that the hardware's check of a buffer's end refuses.
__global__ __launch_bounds__(kThreads) void k_ffn_pack(const uint16_t* from, int64_t ld, uint16_t* to, int64_t ldt, int64_t rows,
                                                       int32_t cols) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int32_t c = int32_t(threadIdx.x) * 8; c < cols; c += kThreads * 8) {
      const CAME8_GLOBAL uint16_t* p = gbl(from) + r * ld + c;
      CAME8_GLOBAL uint16_t* q = gbl(to) + r * ldt + c;
      if (c + 8 <= cols) {
        *(CAME8_GLOBAL u32x4*)q = *(const CAME8_GLOBAL u32x4u*)p;
      } else {
        for (int e = 0; c + e < cols; ++e) q[e] = p[e];
      }
    }
}

}  // namespace came8
