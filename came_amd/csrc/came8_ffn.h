// Matrix-product kernels of the gated feed-forward block for gfx950: C = A B^T over tiles held in registers, with the
// block's elementwise parts in the products' epilogues.
//
// One kernel serves all products of the block and its gradients.  Either operand lies in memory with the summed index
// contiguous ("rows") or with the other one contiguous ("columns"); a thread that loads columns transposes its small
// block in registers on the way to LDS, so no product needs a transposed copy of a weight or an activation.
#pragma once

#include <type_traits>

#include "came8_device.h"
#include "came8_view.h"

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

// The hardware's exponential and reciprocal, a unit in the last place each: accurate ones and their divisions were as long
// as the products (the backward epilogue 1135 us for 8192 by 11008 hidden values, 640 us of it the product).  The error, a
// few 2^-24 of |g|, is that of one more term in the sums that g comes from.
__device__ __forceinline__ float exp_hw(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + exp_hw(-g)); }

// act(g) and, with SLOPE, its derivative, of four values
template <bool SLOPE>
__device__ __forceinline__ void activate(const float (&g)[4], int act, float (&value)[4], float (&slope)[4]) {
  if (act == kSilu) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float s = sigmoid(g[e]);
      value[e] = g[e] * s;
      if (SLOPE) slope[e] = s * (1.0f + g[e] * (1.0f - s));
    }
  } else if (act == kGelu) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float c = 0.5f * (1.0f + erff(g[e] * 0.70710678118654752f));
      value[e] = g[e] * c;
      if (SLOPE) slope[e] = c + g[e] * exp_hw(-0.5f * g[e] * g[e]) * 0.39894228040143268f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // 0.5 (1 + tanh(x)) = sigmoid(2 x)
      const float k = 2.0f * 0.79788456080286536f, gg = g[e] * g[e];
      const float s = sigmoid(k * (g[e] + 0.044715f * gg * g[e]));
      value[e] = g[e] * s;
      const float q = s * (1.0f - s);  // 0 long before gg overflows
      if (SLOPE) slope[e] = s + (q > 0.0f ? g[e] * q * k * (1.0f + 3.0f * 0.044715f * gg) : 0.0f);
    }
  }
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
  int32_t splits;   // workgroups that share a tile's sum
  float* part;      // splits > 1: their sums, [splits][M][N up to a multiple of 4] (kGate: gate and up after each other in
                    // a row), for k_ffn_join; else null
  int32_t act;
  void* out;        // kStore: C; kGate: h; kBack: dg
  int64_t ldo;
  void* out2;       // kBack: du
  void* out3;       // kBack: h, or null
  float* g;         // kGate: where to keep g and u (null: not kept); kBack: where they are kept
  float* u;
  int64_t ldg;
};

// A tile's view of an operand from its next k on: reads past the matrix's end give zeros, whatever the tile.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr uint32_t kNowhere = 0x80000000u;  // an offset past every view's end (offsets within one stay below 2^31)
struct View {
  const char* p;
  int64_t left;  // bytes to the matrix's end, below 1 past it
  int64_t step;  // bytes to the next k step
  int32_t ld;    // bytes from a row (or k) to the next

  __device__ __forceinline__ Buffer buffer() const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, buffer_bytes(left), 0x00027000);
  }
  __device__ __forceinline__ void next(int64_t steps = 1) {
    p += step * steps;
    left -= step * steps;
  }
};

constexpr int kChunkBytes = 16;
constexpr int kRowBytes = 128;  // of a tile in LDS: 8 chunks, 64 (fp32: 32) values of k

// Chunk c of row r lies at place c ^ swz(r) of its row.  A 16-byte read takes 16 lanes at a time, and not in order: lanes 0-3,
// 12-15, 20-23 and 24-27 go together (and 4-11, 16-19, 28-31).  With a fragment's lanes, row l % 16 and chunk l / 16, these
// are 16 different places of two rows' length, all 64 banks once; eight lanes that write a chunk of rows 8 apart (columns on
// their way in) touch eight places.  (With places that only 8 lanes in order tell apart, every read took twice its time.)
// By the counters, launches of rows alone have conflicts in 0 to 1% of their LDS cycles, those with columns, whose writes are 8
// bytes a lane in tiles of 256, in 24% (the gradients) and 16% (dy Wd): 8192 tokens of 4096 and 11008 in bf16.
// swz is linear: of rows whose bits do not overlap it is the exclusive or.
__host__ __device__ constexpr int swz(int r) { return (r >> 3 & 1) | ((r ^ r >> 4) & 2) | ((r ^ r >> 1 ^ r >> 2) & 4); }

// ------------------------------------------------------------------------------------------------ operands' way in
// R rows by 8 chunks of k, NT threads: 16-byte loads into registers (fetch), later written to LDS (put).
//
// Rows: a thread loads chunk t % 8 of every NT / 8-th row from row t / 8 on; a chunk at or past k = K lies nowhere and gives
// zeros (a chunk that K cuts holds zeros in memory).  Columns: a thread loads kLoads successive k of kVec rows, and k past K
// lie past the end.  HALF > 0: rows taken in turns of HALF from two matrices (the gate's and the up projection's weights);
// loads i of a thread go to the one and the other in turn.  ODD: 16-bit rows an odd number of elements apart, every other
// one of which starts in the middle of a word: the words that hold a chunk are loaded, five of them, and shifted on their way
// to LDS, where a chunk that K cuts loses what is of the next row.
template <typename T, int R, int NT, bool ROWS, int HALF = 0, bool ODD = false>
struct Stage {
  static constexpr int kElem = int(sizeof(typename T::storage));
  static constexpr int kVec = kChunkBytes / kElem;        // elements of a chunk
  static constexpr int kLoads = R * 8 / NT;               // 16-byte loads a thread
  static constexpr int kStep = NT / 8;                    // rows: from a load's to the next
  static_assert(!ODD || (ROWS && HALF == 0 && kElem == 2 && kStep % 2 == 0), "");
  u32x4 v[kLoads];
  uint32_t fifth[ODD ? kLoads : 1], shift;  // ODD: 2 where the thread's rows start in the middle of a word
  int odd_left;

  // left: K less the view's first k
  __device__ __forceinline__ void fetch(const View& a, const View& a1, int left) {
    const uint32_t t = threadIdx.x;
    if constexpr (!ROWS) {
      const Buffer buf = a.buffer();
      const uint32_t off = t / (R / kVec) * kLoads * a.ld + t % (R / kVec) * kChunkBytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(buf, off + i * a.ld, 0, 0);
    } else {
      const bool out = int(t & 7) * kVec >= left;
      const Buffer buf = a.buffer();
      const uint32_t off = out ? kNowhere : (t >> 3) * a.ld + (t & 7) * kChunkBytes;
      if constexpr (ODD) {
        shift = off & 2;
        odd_left = left;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          v[i] = __builtin_amdgcn_raw_buffer_load_b128(buf, off - shift + i * kStep * a.ld, 0, 0);
          fifth[i] = __builtin_amdgcn_raw_buffer_load_b32(buf, off - shift + i * kStep * a.ld + 16, 0, 0);
        }
      } else if constexpr (HALF == 0) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(buf, off + i * kStep * a.ld, 0, 0);
      } else {
        const Buffer buf1 = a1.buffer();
        const uint32_t off1 = out ? kNowhere : (t >> 3) * a1.ld + (t & 7) * kChunkBytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          v[i] = (i & 1) ? __builtin_amdgcn_raw_buffer_load_b128(buf1, off1 + i / 2 * kStep * a1.ld, 0, 0)
                         : __builtin_amdgcn_raw_buffer_load_b128(buf, off + i / 2 * kStep * a.ld, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void put(char* lds) const {
    const int t = int(threadIdx.x);
    if constexpr (ROWS) {
      constexpr int H = HALF == 0 ? kStep : HALF;
      // the first load's row; load i's is `row` further
      const int c = t & 7, r = HALF == 0 ? t >> 3 : (t >> 3) / H * 2 * H + (t >> 3) % H;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = HALF == 0 ? i * kStep : i / 2 * 2 * kStep + (i & 1) * HALF;
        if constexpr (ODD) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_alignbyte(e < 3 ? v[i][e + 1] : fifth[i], v[i][e], shift);
          if (odd_left < (c + 1) * kVec) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = c * kVec + 2 * e;
              w[e] = k + 1 < odd_left ? w[e] : k < odd_left ? w[e] & 0xffffu : 0u;
            }
          }
          *reinterpret_cast<u32x4*>(lds + (r * kRowBytes + ((c ^ swz(r)) ^ swz(row)) * kChunkBytes) + row * kRowBytes) = w;
          continue;
        }
        *reinterpret_cast<u32x4*>(lds + (r * kRowBytes + ((c ^ swz(r)) ^ swz(row)) * kChunkBytes) + row * kRowBytes) = v[i];
      }
    } else if constexpr (kElem == 4) {
      const int r = (t % (R / kVec)) * kVec, k = (t / (R / kVec)) * kLoads;  // first row, first k
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kLoads >= 4) {
#pragma unroll
          for (int c = 0; c < kLoads / 4; ++c)
            *reinterpret_cast<u32x4*>(lds + (r + e) * kRowBytes + (((k / 4 + c) ^ swz(r + e)) * kChunkBytes)) =
                u32x4{v[4 * c][e], v[4 * c + 1][e], v[4 * c + 2][e], v[4 * c + 3][e]};
        } else {
          *reinterpret_cast<u32x2*>(lds + (r + e) * kRowBytes + (((k / 4) ^ swz(r + e)) * kChunkBytes) + (k % 4) * 4) =
              u32x2{v[0][e], v[1][e]};
        }
      }
    } else {
      const int r = (t % (R / kVec)) * kVec, k = (t / (R / kVec)) * kLoads;
      // v[j] word w holds rows 2w, 2w + 1 of k + j: halves of two words make one word of a row
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t w[kLoads / 2];
#pragma unroll
        for (int j = 0; j < kLoads / 2; ++j)
          w[j] = __builtin_amdgcn_perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
        char* at = lds + (r + e) * kRowBytes + (((k / 8) ^ swz(r + e)) * kChunkBytes) + (k % 8) * 2;
        if constexpr (kLoads == 8) *reinterpret_cast<u32x4*>(at) = u32x4{w[0], w[1], w[2], w[3]};
        else if constexpr (kLoads == 4) *reinterpret_cast<u32x2*>(at) = u32x2{w[0], w[1]};
        else *reinterpret_cast<uint32_t*>(at) = w[0];
      }
    }
  }
};

// fp32 values as three bf16 ones, each the rounding of what the ones before leave: their sum is the value to 2^-24 of it.
//
// LARGE: for values of any size.  The first part is bounded by bf16's largest value, so that a value that would round to infinity
// leaves a rest.  An infinity is its sign, zero and itself: the third part meets the other operand's first alone, which has the
// other's sign and is zero where that is (and below 2^-134), and the sign meets what is finite where the other operand is, so no
// part of it cancels the infinity.  NaN gets to the third part as well.  Without LARGE no part is bounded: a thread looks
// over its loads once (2048 tokens of 4096 and 11008 forward and backward 8.98 ms, 9.97 with every value bounded).
constexpr float kLargestBf16 = 0x1.fep127f;
struct Parts {
  uint32_t w[3];  // of two values, packed
};
template <bool LARGE>
__device__ __forceinline__ Parts parts_of(float x, float y) {
  auto first = [](float v) {
    if (!LARGE) return v;
    const float most = __builtin_isinf(v) ? 1.0f : kLargestBf16;
    return __builtin_amdgcn_fmed3f(v, -most, most);
  };
  auto second = [](float v) { return LARGE && __builtin_isinf(v) ? 0.0f : v; };
  Parts p;
  p.w[0] = uint32_t(BF16::store(first(x))) | uint32_t(BF16::store(first(y))) << 16;
  x -= BF16::elem(&p.w[0], 0);
  y -= BF16::elem(&p.w[0], 1);
  p.w[1] = uint32_t(BF16::store(second(x))) | uint32_t(BF16::store(second(y))) << 16;
  x -= BF16::elem(&p.w[1], 0);
  y -= BF16::elem(&p.w[1], 1);
  p.w[2] = uint32_t(BF16::store(x)) | uint32_t(BF16::store(y)) << 16;
  return p;
}

// the largest magnitude of a thread's loads and `top`; NaN if there is one
template <int R, int NT, bool ROWS, int HALF>
__device__ __forceinline__ float largest(const Stage<F32, R, NT, ROWS, HALF>& s, float top) {
#pragma unroll
  for (int i = 0; i < Stage<F32, R, NT, ROWS, HALF>::kLoads; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __builtin_elementwise_maximum(top, __builtin_fabsf(__uint_as_float(s.v[i][e])));
  return top;
}

// Rows of three parts in LDS: 64 bytes each, 32 values of k.  Chunk c of row r lies at c ^ part_swz(r), so that the lanes of a
// read (see swz) touch all banks once.
constexpr int kPartBytes = 64, kPartRow = 3 * kPartBytes;
__host__ __device__ constexpr int part_swz(int r) { return (4 - (r >> 2 & 3)) & 3; }

// Stage::put for rows of parts
template <bool LARGE, int R, int NT, bool ROWS, int HALF>
__device__ __forceinline__ void put_parts(const Stage<F32, R, NT, ROWS, HALF>& s, char* lds) {
  using St = Stage<F32, R, NT, ROWS, HALF>;
  const int t = int(threadIdx.x);
  if constexpr (ROWS) {
    constexpr int H = HALF == 0 ? St::kStep : HALF;
    const int c = t & 7, r = HALF == 0 ? t >> 3 : (t >> 3) / H * 2 * H + (t >> 3) % H;
#pragma unroll
    for (int i = 0; i < St::kLoads; ++i) {
      const int row = r + (HALF == 0 ? i * St::kStep : i / 2 * 2 * St::kStep + (i & 1) * HALF);
      const Parts a = parts_of<LARGE>(__uint_as_float(s.v[i][0]), __uint_as_float(s.v[i][1]));
      const Parts b = parts_of<LARGE>(__uint_as_float(s.v[i][2]), __uint_as_float(s.v[i][3]));
      char* at = lds + row * kPartRow + ((c >> 1) ^ part_swz(row)) * kChunkBytes + (c & 1) * 8;
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x2*>(at + p * kPartBytes) = u32x2{a.w[p], b.w[p]};
    }
  } else {
    const int r = (t % (R / 4)) * 4, k = (t / (R / 4)) * St::kLoads;  // first row, first k
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      char* at = lds + (r + e) * kPartRow + ((k >> 3) ^ part_swz(r + e)) * kChunkBytes + (k & 7) * 2;
      const Parts a = parts_of<LARGE>(__uint_as_float(s.v[0][e]), __uint_as_float(s.v[1][e]));
      if constexpr (St::kLoads == 4) {
        const Parts b = parts_of<LARGE>(__uint_as_float(s.v[2][e]), __uint_as_float(s.v[3][e]));
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x2*>(at + p * kPartBytes) = u32x2{a.w[p], b.w[p]};
      } else {
        static_assert(St::kLoads == 2, "");
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint32_t*>(at + p * kPartBytes) = a.w[p];
      }
    }
  }
}

// V consecutive values to a row of N elements at any address, those past N left out (unless the row is padded past it)
template <typename T>
__device__ __forceinline__ void store4(void* row, int n, int N, const float (&x)[4]) {
  using S = typename T::storage;
  CAME8_GLOBAL S* p = gbl(static_cast<S*>(row)) + n;
  if (n + 4 <= N) {
    if constexpr (sizeof(S) == 4)
      *(CAME8_GLOBAL f32x4u*)p = f32x4u{x[0], x[1], x[2], x[3]};
    else
      *(CAME8_GLOBAL u32x2u*)p = u32x2u{uint32_t(T::store(x[0])) | uint32_t(T::store(x[1])) << 16,
                                        uint32_t(T::store(x[2])) | uint32_t(T::store(x[3])) << 16};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) p[e] = T::store(x[e]);
  }
}

__device__ __forceinline__ void load4(const float* row, int n, int N, float (&x)[4]) {
  const CAME8_GLOBAL float* p = gbl(row) + n;
  if (n + 4 <= N) {
    const f32x4u v = *(const CAME8_GLOBAL f32x4u*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = n + e < N ? p[e] : 0.0f;
  }
}

// dg, du and h of four values, from dh, g and u (zeros past N, where rows are padded)
template <typename T>
__device__ __forceinline__ void store_back(const GemmArgs& args, int64_t row, int n, const float (&dh)[4], const float (&g)[4],
                                           const float (&u)[4]) {
  using S = typename T::storage;
  float h[4], dg[4], du[4];
  activate<true>(g, args.act, h, dg);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool in = n + e < args.N;  // past N dh is of no column, and may hold anything
    du[e] = in ? dh[e] * h[e] : 0.0f;
    dg[e] = in ? dg[e] * (dh[e] * u[e]) : 0.0f;
    h[e] = in ? h[e] * u[e] : 0.0f;
  }
  const int ld = int(args.ldo);
  store4<T>(static_cast<S*>(args.out) + row * args.ldo, n, ld, dg);
  store4<T>(static_cast<S*>(args.out2) + row * args.ldo, n, ld, du);
  if (args.out3) store4<T>(static_cast<S*>(args.out3) + row * args.ldo, n, ld, h);
}

// h of four values of g and u (zeros past N, where rows are padded), and g and u where they are kept
template <typename T>
__device__ __forceinline__ void store_gate(const GemmArgs& args, int64_t row, int n, const float (&g)[4], const float (&u)[4]) {
  float h[4], none[4];
  activate<false>(g, args.act, h, none);
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = n + e < args.N ? h[e] * u[e] : 0.0f;
  store4<T>(static_cast<typename T::storage*>(args.out) + row * args.ldo, n, int(args.ldo), h);
  if (args.g) {
    store4<F32>(args.g + row * args.ldg, n, args.N, g);
    store4<F32>(args.u + row * args.ldg, n, args.N, u);
  }
}

// ------------------------------------------------------------------------------------------------------ product
// Asks the scheduler to spread `count` instructions of the given kinds evenly among `products` matrix instructions, and to
// move nothing past the end of the phase.
constexpr int kMfma = 0x008, kVmemRead = 0x020, kDsRead = 0x100, kDsWrite = 0x200;
template <int KINDS, int COUNT, int PRODUCTS, int K = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (K < COUNT) {
    __builtin_amdgcn_sched_group_barrier(kMfma, PRODUCTS * (K + 1) / COUNT - PRODUCTS * K / COUNT, 0);
    __builtin_amdgcn_sched_group_barrier(KINDS, 1, 0);
    interleave<KINDS, COUNT, PRODUCTS, K + 1>();
  } else {
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The tiles: B by B on 2 by WAVES_N wavefronts, and for fp32 at B = 256 ("parts") 256 by 128 on 4 by 2.
template <typename T, int B, int WAVES_N>
struct Tile {
  static constexpr bool kParts = std::is_same<T, F32>::value && B == 256;
  static constexpr int kWavesM = kParts ? 4 : 2, kWidth = kParts ? 128 : B, kGroup = kWavesM * WAVES_N * kWave;
  static constexpr int kBytes = (B + kWidth) * (kParts ? kPartRow : kRowBytes);  // of a step's operands
};

// Workgroups of 2 by WAVES_N wavefronts on a tile of BM by BN; an accumulator lane holds 4 consecutive columns of a row.
// kGate: the tile's BN rows of weights are, in turns of half a wavefront's, gate and up projection, so that a wavefront
// holds both values of its columns of h.
//
// Step t of k is four phases, each of a quarter of its products, with the LDS reads of the next phase among them; in the second
// the operands of step t + 1 go from registers to the other LDS buffer, and those of step t + 2 are loaded.  The step's one
// barrier stands before the last phase, whose reads are the first of step t + 1.  So neither LDS reads nor global loads are
// waited for at the barrier.  Steps past the end load zeros.
//
// fp32 at BM = 256: the matrix instructions of fp32 run at a sixteenth of bf16's rate.  The operands are taken apart into three
// bf16 parts on their way to LDS, and the six products of parts down to 2^-16 of the largest, summed in fp32, are a product
// of fp32's accuracy at a sixth of bf16's rate: 2048 tokens of 4096 and 11008 forward and backward 9.0 ms (185
// TFLOP/s) against 12.4.
template <typename T, int BM, int WAVES_N, bool AROWS, bool BROWS, Epilogue EPI, bool ODD = false>
__device__ __forceinline__ void product(const GemmArgs& args, int b, char* lds) {
  using S = typename T::storage;
  using Shape = Tile<T, BM, WAVES_N>;
  constexpr int kElem = int(sizeof(S));
  constexpr int BK = kRowBytes / kElem;
  constexpr int BN = Shape::kWidth, WAVES_M = Shape::kWavesM, NT = Shape::kGroup;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
  constexpr int kTileBytes = Shape::kBytes;

  // Workgroups go to the 8 XCDs in turn: each XCD gets a run of successive tiles, 8 tiles of rows by the columns.
  int tm, tn, split;
  {
    const int tiles = args.tiles_m * args.tiles_n, all = tiles * args.splits;
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
  const int m0 = tm * BM, n0 = tn * (EPI == kGate ? BN / 2 : BN);
  const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
  const int wm = wave % WAVES_M, wn = wave / WAVES_M;

  // Steps loaded ahead; step t is in registers t % D.  Two where registers allow: 1021 tokens of 1024 and 2731 in fp32, tiles
  // of 64 and 128, 516 us with one and 492 with two, 32 tokens of 4096 and 11008 in bf16 80 and 75 us (with sums in
  // up to 16 shares).
  constexpr int D = BM < 256 ? 2 : 1;
  Stage<T, BM, NT, AROWS> sa[D];
  Stage<T, BN, NT, BROWS, EPI == kGate ? WN / 2 : 0, ODD> sb[D];
  const int steps = (args.K + BK - 1) / BK;
  const int every = steps * args.nseg;
  int ahead = int(int64_t(every) * split / args.splits);  // the step that is fetched next
  const int total = int(int64_t(every) * (split + 1) / args.splits) - ahead;
  auto view = [&](const Operand& o, bool rows, int at, int extent) {
    const int64_t ld = o.ld * kElem;
    View v;
    v.p = static_cast<const char*>(o.p) + (rows ? at * ld : int64_t(at) * kElem);
    v.left = view_bytes(rows, extent - at, args.K, ld, kElem);
    v.step = rows ? kRowBytes : BK * ld;
    v.ld = int32_t(ld);
    return v;
  };
  View va = view(args.seg[0].a, AROWS, m0, args.M), vb = view(args.seg[0].b, EPI == kGate || BROWS, n0, args.N);
  // the second segment's (kGate: the up projection's weights)
  const View va1 = args.nseg > 1 ? view(args.seg[1].a, AROWS, m0, args.M) : va;
  View vb1 = EPI == kGate ? view(args.b2, true, n0, args.N) : args.nseg > 1 ? view(args.seg[1].b, BROWS, n0, args.N) : vb;
  if (EPI != kGate && ahead >= steps && args.nseg > 1) {
    va = va1;
    vb = vb1;
  }
  int left = args.K - (ahead % steps) * BK;  // K less the next step's first k
  va.next(ahead % steps);
  vb.next(ahead % steps);
  if (EPI == kGate) vb1.next(ahead);
  auto fetch = [&](int slot) __attribute__((always_inline)) {
    sa[slot].fetch(va, va, left);
    sb[slot].fetch(vb, vb1, left);
    va.next();
    vb.next();
    left -= BK;
    if constexpr (EPI == kGate) {
      vb1.next();
    } else {
      const bool turn = ++ahead == steps && args.nseg > 1;
      va.p = turn ? va1.p : va.p;
      va.left = turn ? va1.left : va.left;
      va.step = turn ? va1.step : va.step;
      va.ld = turn ? va1.ld : va.ld;
      vb.p = turn ? vb1.p : vb.p;
      vb.left = turn ? vb1.left : vb.left;
      vb.step = turn ? vb1.step : vb.step;
      vb.ld = turn ? vb1.ld : vb.ld;
      left = turn ? args.K : left;
    }
  };
  f32x4 acc[FM][FN] = {};
  if constexpr (Shape::kParts) {
    fetch(0);
    for (int t = 0; t < total; ++t) {
      char* at = lds + (t & 1) * kTileBytes;
      const bool large = !(largest(sb[0], largest(sa[0], 0.0f)) <= kLargestBf16);
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(large) == 0, 1)) {
        put_parts<false>(sa[0], at);
        put_parts<false>(sb[0], at + BM * kPartRow);
      } else {
        put_parts<true>(sa[0], at);
        put_parts<true>(sb[0], at + BM * kPartRow);
      }
      fetch(0);
      __syncthreads();  // the other buffer's last reads are behind every wavefront that has come here
      const int r = lane % 16, place = r * kPartRow + (lane / 16 ^ part_swz(r)) * kChunkBytes;
      const char* pa = at + wm * WM * kPartRow + place;
      const char* pb = at + (BM + wn * WN) * kPartRow + place;
      u32x4 fb[3][FN];
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[p][j] = *reinterpret_cast<const u32x4*>(pb + j * 16 * kPartRow + p * kPartBytes);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        u32x4 fa[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) fa[p] = *reinterpret_cast<const u32x4*>(pa + i * 16 * kPartRow + p * kPartBytes);
#pragma unroll
        for (int p = 2; p >= 0; --p)  // the smallest products first
#pragma unroll
          for (int q = 2 - p; q >= 0; --q)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma_chunk<BF16>(fb[q][j], fa[p], acc[i][j]);
      }
    }
  } else {
    auto put = [&](int t, int slot) __attribute__((always_inline)) {
      char* to = lds + (t & 1) * kTileBytes;
      sa[slot].put(to);
      sb[slot].put(to + BM * kRowBytes);
    };
    // Fragment i of half s: row 16 i + lane % 16 of the wavefront's, chunk 4 s + lane / 16, at place
    // (lane / 16) ^ swz(the wavefront's first row + lane % 16) ^ 4 s ^ swz(16 i), one of four that differ by 2 v.
    const int fr = lane % 16;
    uint32_t pa[4], pb[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      pa[v] = uint32_t((wm * WM + fr) * kRowBytes + (lane / 16 ^ swz(wm * (WM % 64) + fr) ^ (2 * v)) * kChunkBytes);
      pb[v] = uint32_t((BM + wn * WN + fr) * kRowBytes + (lane / 16 ^ swz(wn * (WN % 64) + fr) ^ (2 * v)) * kChunkBytes);
    }
    u32x4 lo[FM / 2], hi[FM / 2], fb[2][FN];
    auto read_a = [&](u32x4(&f)[FM / 2], int t, int s, int i0) __attribute__((always_inline)) {
      const char* a = lds + (t & 1) * kTileBytes;
#pragma unroll
      for (int i = 0; i < FM / 2; ++i)
        f[i] = *reinterpret_cast<const u32x4*>(a + pa[(4 * s ^ swz(16 * (i0 + i))) / 2] + (i0 + i) * 16 * kRowBytes);
    };
    auto read_b = [&](int t, int s, int j0) __attribute__((always_inline)) {
      const char* b = lds + (t & 1) * kTileBytes;
#pragma unroll
      for (int j = j0; j < j0 + FN / 2; ++j)
        fb[s][j] = *reinterpret_cast<const u32x4*>(b + pb[(4 * s ^ swz(16 * j)) / 2] + j * 16 * kRowBytes);
    };

    auto multiply = [&](const u32x4(&f)[FM / 2], int s, int i0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < FM / 2; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i0 + i][j] = mfma_chunk<T>(fb[s][j], f[i], acc[i0 + i][j]);
    };
    constexpr int kProducts = FM / 2 * FN * (kElem == 4 ? 4 : 1);  // of a phase
    // Step t + 2 is loaded as soon as step t + 1 has left the registers, a whole step before its use (8192 tokens forward and
    // backward 6555 us with loads half a step ahead, 6452 so); with columns, whose way to LDS takes registers, a quarter later.
    constexpr bool kEarly = AROWS && BROWS;
    fetch(0);
    put(0, 0);
#pragma unroll
    for (int d = 1; d <= D; ++d) fetch(d % D);
    __syncthreads();
    read_a(lo, 0, 0, 0);
    read_b(0, 0, 0);
    read_b(0, 0, FN / 2);
    auto step = [&](int t, int slot) __attribute__((always_inline)) {  // slot: of step t + 1
      read_a(hi, t, 0, FM / 2);
      read_b(t, 1, 0);
      read_b(t, 1, FN / 2);
      multiply(lo, 0, 0);
      interleave<kDsRead, FM / 2 + FN, kProducts>();
      read_a(lo, t, 1, 0);
      put(t + 1, slot);
      if constexpr (kEarly) fetch(slot);
      multiply(hi, 0, FM / 2);
      interleave<kDsRead | kDsWrite | kVmemRead, FM / 2 + FM + FN + (kEarly ? 8 : 0), kProducts>();
      read_a(hi, t, 1, FM / 2);
      if constexpr (!kEarly) fetch(slot);
      multiply(lo, 1, 0);
      interleave<kDsRead | kVmemRead, FM / 2 + (kEarly ? 0 : 8), kProducts>();
      // every wavefront has read its last of step t, whose place the next put takes, and written its part of step t + 1
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      read_a(lo, t + 1, 0, 0);
      read_b(t + 1, 0, 0);
      read_b(t + 1, 0, FN / 2);
      multiply(hi, 1, FM / 2);
      interleave<kDsRead, FM / 2 + FN, kProducts>();
    };
    for (int t = 0; t < total; t += D)
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (d == 0 || t + d < total) step(t + d, (d + 1) % D);
  }

  // acc[i][j][e]: row 16 i + lane % 16 of the wavefront's, column 16 j + 4 (lane / 16) + e.  Up to 64 rows at a time go
  // through the wavefront's own part of LDS, so that lanes of successive columns read and write memory together; chunk c of
  // row r lies at c ^ r.  Several rounds' reads of g and u are in flight before the first is used.
  constexpr int kPart = FM < 4 ? FM : 4;
  constexpr int kChunks = WN / 4;
  static_assert(WAVES_M * WAVES_N * kPart * 16 * WN * 4 <= 2 * kTileBytes, "");
  char* mine = lds + wave * (kPart * 16 * WN * 4);
  constexpr int kCols = EPI == kGate ? WN / 2 : WN;  // of the output
  constexpr int kLanes = kCols / 4, kRows = kWave / kLanes, kRounds = kPart * 16 / kRows;
  constexpr int kBatch = kRounds < 4 ? kRounds : 4;
  const int cc = lane % kLanes, r0 = lane / kLanes, n = n0 + wn * kCols + cc * 4;
  auto slot = [&](int r, int c) { return reinterpret_cast<f32x4*>(mine + r * (WN * 4) + ((c ^ r) & (kChunks - 1)) * 16); };
  float gn[kBatch][4] = {}, un[kBatch][4] = {};  // of the next rounds
  __syncthreads();
#pragma unroll
  for (int part = 0; part < FM / kPart; ++part) {
#pragma unroll
    for (int i = 0; i < kPart; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) *slot(i * 16 + lane % 16, j * 4 + lane / 16) = acc[part * kPart + i][j];
    const int m1 = m0 + wm * WM + part * kPart * 16 + r0;
    auto load = [&](int q) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int m = m1 + (q + k) * kRows;
        if (m < args.M) {
          load4(args.g + int64_t(m) * args.ldg, n, args.N, gn[k]);
          load4(args.u + int64_t(m) * args.ldg, n, args.N, un[k]);
        }
      }
    };
    if (EPI == kBack && args.part == nullptr) load(0);
#pragma unroll 1
    for (int q = 0; q < kRounds; q += kBatch) {
      const int m = m1 + q * kRows;
      float g[kBatch][4], u[kBatch][4];
      if (EPI == kBack && args.part == nullptr) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            g[k][e] = gn[k][e];
            u[k][e] = un[k][e];
          }
        if (q + kBatch < kRounds) load(q + kBatch);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = (q + k) * kRows + r0;
        if (m + k * kRows >= args.M) continue;
        const int64_t row = m + k * kRows;
        const f32x4 c = *slot(r, cc);
        if (args.part) {
          const int pitch = (args.N + 3) & ~3;
          float* to = args.part + (int64_t(split) * args.M + row) * pitch * (EPI == kGate ? 2 : 1);
          store4<F32>(to, n, pitch, {c[0], c[1], c[2], c[3]});
          if constexpr (EPI == kGate) {
            const f32x4 d = *slot(r, cc + kChunks / 2);
            store4<F32>(to + pitch, n, pitch, {d[0], d[1], d[2], d[3]});
          }
          continue;
        }
        S* out = static_cast<S*>(args.out) + row * args.ldo;
        if constexpr (EPI == kStore) {
          store4<T>(out, n, args.N, {c[0], c[1], c[2], c[3]});
        } else if constexpr (EPI == kGate) {
          const f32x4 d = *slot(r, cc + kChunks / 2);
          store_gate<T>(args, row, n, {c[0], c[1], c[2], c[3]}, {d[0], d[1], d[2], d[3]});
        } else {
          store_back<T>(args, row, n, {c[0], c[1], c[2], c[3]}, g[k], u[k]);
        }
      }
    }
  }
}

template <typename T, int B, int WAVES_N, bool AROWS, bool BROWS, Epilogue EPI, bool ODD>
__global__ __launch_bounds__((Tile<T, B, WAVES_N>::kGroup), 2) void k_ffn_gemm(const GemmArgs args) {
  __shared__ __attribute__((aligned(16))) char lds[2 * Tile<T, B, WAVES_N>::kBytes];
  product<T, B, WAVES_N, AROWS, BROWS, EPI, ODD>(args, int(blockIdx.x), lds);
}

// The products that only wait for dg, du and h: dx and the weights' gradients, one launch, the longest sums first.  The last
// tiles of one fill the CUs beside the first of the next.
struct GradArgs {
  GemmArgs dx;
  GemmArgs dw[3];
  int32_t first[4];  // workgroups before each dw, and all
};
template <typename T, int B, int WAVES_N>
__global__ __launch_bounds__((Tile<T, B, WAVES_N>::kGroup), 2) void k_ffn_grads(const GradArgs args) {
  __shared__ __attribute__((aligned(16))) char lds[2 * Tile<T, B, WAVES_N>::kBytes];
  const int b = int(blockIdx.x);
  if (b < args.first[0]) {
    product<T, B, WAVES_N, true, false, kStore>(args.dx, b, lds);
  } else {
    const int k = (b >= args.first[1]) + (b >= args.first[2]);
    product<T, B, WAVES_N, false, false, kStore>(args.dw[k], b - args.first[k], lds);
  }
}

// The shares of tiles whose sums were split, added in order, and the epilogue.
template <typename T, Epilogue EPI>
__device__ __forceinline__ void join(const GemmArgs& args) {
  const int pitch = (args.N + 3) & ~3, quads = pitch / 4;
  const int64_t width = int64_t(pitch) * (EPI == kGate ? 2 : 1), all = int64_t(args.M) * quads;
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < all; i += int64_t(gridDim.x) * kThreads) {
    const int64_t row = i / quads;
    const int n = int(i - row * quads) * 4;
    const CAME8_GLOBAL float* part = gbl(args.part) + row * width + n;
    f32x4 sum = {}, sum1 = {};
#pragma unroll 4
    for (int s = 0; s < args.splits; ++s, part += args.M * width) {
      sum += *(const CAME8_GLOBAL f32x4*)part;
      if (EPI == kGate) sum1 += *(const CAME8_GLOBAL f32x4*)(part + pitch);
    }
    const float x[4] = {sum[0], sum[1], sum[2], sum[3]};
    const float none[4] = {};
    // and the padded end of the row, where it is more than a quad past N
    const int end = n + 4 == pitch ? int(args.ldo) : 0;
    if constexpr (EPI == kStore) {
      store4<T>(static_cast<typename T::storage*>(args.out) + row * args.ldo, n, args.N, x);
    } else if constexpr (EPI == kGate) {
      store_gate<T>(args, row, n, x, {sum1[0], sum1[1], sum1[2], sum1[3]});
      for (int p = pitch; p < end; p += 4) store4<T>(static_cast<typename T::storage*>(args.out) + row * args.ldo, p, end, none);
    } else {
      float g[4], u[4];
      load4(args.g + row * args.ldg, n, args.N, g);
      load4(args.u + row * args.ldg, n, args.N, u);
      store_back<T>(args, row, n, x, g, u);
      for (int p = pitch; p < end; p += 4) store_back<T>(args, row, p, none, none, none);
    }
  }
}

template <typename T, Epilogue EPI>
__global__ __launch_bounds__(kThreads) void k_ffn_join(const GemmArgs args) {
  join<T, EPI>(args);
}

// Of dx and the weights' gradients, those that were split: blockIdx.y says which.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_ffn_join_grads(const GradArgs args) {
  const GemmArgs& g = blockIdx.y == 0 ? args.dx : args.dw[blockIdx.y - 1];
  if (g.part) join<T, kStore>(g);
}

// ------------------------------------------------------------------------------------------------- few rows of x
// Up to 16 rows: the weights are read once and are all there is to wait for, so no tile goes through LDS.  A workgroup has
// 16 rows of the weights (kGate: of both) and all rows of x; its 8 wavefronts take steps of 128 bytes of k in turn, a lane
// two chunks of a row at once, whole lines of a row by four lanes, four steps in flight; their sums are added in order in
// LDS.  Rows may start at any element.  One token of 4096 and 11008 in bf16: 36.8 us for 180 MB of gate and up, 22 for the
// 90 MB of down (4.9 and 4.1 TB/s), 60 together, 75 in tiles; 2 or 8 steps in flight and 16 wavefronts changed nothing.  With
// 32 rows it took 89 us, tiles 66: x then costs more loads than the weights.
//
// h between the two is kept in fp32: as an operand it is its rounding to the type and the rest's, two products with sums of
// their own, which the weights' way hides, so that y is rounded once.  What the type rounds to infinity is infinite there too.
struct FewArgs {
  const void* x;     // down: h, float
  int64_t ldx;
  const void* w[2];  // kGate: gate and up
  int64_t ldw[2];
  int32_t M, N, K, act;
  void* out;         // gate and up: h, float
  int64_t ldo;
  float* g;
  float* u;
  int64_t ldg;
};
constexpr int kFewRows = 16;

// a chunk at any address its type allows
typedef uint32_t u32x4w __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
using AnyChunk = typename std::conditional<sizeof(typename T::storage) == 4, u32x4w, u32x4u>::type;

// chunk at k of a row of K elements, what is past K as zeros
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const CAME8_GLOBAL typename T::storage* row, int k, int K) {
  using S = typename T::storage;
  constexpr int V = kChunkBytes / int(sizeof(S));
  if (k + V <= K) return *(const CAME8_GLOBAL AnyChunk<T>*)(row + k);
  u32x4 v = {};
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (k + e < K) {
      if constexpr (sizeof(S) == 4) v[e] = __float_as_uint(row[k + e]);
      else v[e / 2] |= uint32_t(row[k + e]) << (16 * (e & 1));
    }
  return v;
}

// 8 floats as two chunks of a 16-bit type: their roundings, and the roundings of the rest (none of what rounds to infinity)
template <typename T>
__device__ __forceinline__ void split_chunk(f32x4 a, f32x4 b, u32x4& high, u32x4& low) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = i < 2 ? a[2 * i] : b[2 * i - 4], y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
    const uint32_t hx = T::store(x), hy = T::store(y);
    const uint32_t word = hx | hy << 16;
    high[i] = word;
    float rx = x - T::elem(&word, 0), ry = y - T::elem(&word, 1);
    rx = fabsf(rx) <= 0x1p127f ? rx : 0.0f;
    ry = fabsf(ry) <= 0x1p127f ? ry : 0.0f;
    low[i] = uint32_t(T::store(rx)) | uint32_t(T::store(ry)) << 16;
  }
}

template <typename T, bool GATE>
__global__ __launch_bounds__(512) void k_ffn_few(const FewArgs args) {
  using S = typename T::storage;
  using raw = AnyChunk<T>;
  constexpr int V = kChunkBytes / int(sizeof(S)), BK = kRowBytes / int(sizeof(S)), G = GATE ? 2 : 1, NW = 8;
  constexpr int U = 4;  // steps in flight
  constexpr bool kSplit = !GATE && sizeof(S) == 2;  // x is h in fp32, in two 16-bit parts
  constexpr int A = kSplit ? 2 : G;                 // kSplit: sums of h's rounding and of its rest
  __shared__ f32x4 sums[NW][A][kWave];
  const int lane = int(threadIdx.x) % kWave, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int n0 = int(blockIdx.x) * 16, q = lane / 16 * 2 * V;
  const CAME8_GLOBAL S* w[G];  // rows past the end are not stored: any row will do
#pragma unroll
  for (int i = 0; i < G; ++i)
    w[i] = gbl(static_cast<const S*>(args.w[i])) + int64_t(min(n0 + lane % 16, args.N - 1)) * args.ldw[i] + q;
  using X = typename std::conditional<GATE, S, float>::type;
  constexpr int P = kSplit ? 2 : 1;
  const CAME8_GLOBAL X* x = gbl(static_cast<const X*>(args.x)) + int64_t(min(lane % 16, args.M - 1)) * args.ldx + q;

  f32x4 acc[A] = {};
  const int full = args.K / BK;
  for (int s0 = wave; s0 < full; s0 += NW * U) {
    u32x4 wv[U][G][2], xv[U][2][P];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * NW < full) {
        const int64_t k = int64_t(s0 + u * NW) * BK;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int i = 0; i < G; ++i) wv[u][i][c] = __builtin_nontemporal_load((const CAME8_GLOBAL raw*)(w[i] + k + c * V));
#pragma unroll
          for (int p = 0; p < P; ++p) {
            if constexpr (GATE) xv[u][c][p] = *(const CAME8_GLOBAL raw*)(x + k + c * V);
            else xv[u][c][p] = __builtin_bit_cast(u32x4, *(const CAME8_GLOBAL f32x4*)(x + k + c * V + 4 * p));
          }
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * NW < full)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if constexpr (kSplit) {
            u32x4 high, low;
            split_chunk<T>(__builtin_bit_cast(f32x4, xv[u][c][0]), __builtin_bit_cast(f32x4, xv[u][c][1]), high, low);
            acc[0] = mfma_chunk<T>(wv[u][0][c], high, acc[0]);
            acc[1] = mfma_chunk<T>(wv[u][0][c], low, acc[1]);
          } else {
#pragma unroll
            for (int g = 0; g < G; ++g) acc[g] = mfma_chunk<T>(wv[u][g][c], xv[u][c][0], acc[g]);
          }
        }
  }
  if (full * BK < args.K && full % NW == wave) {
    const int k = full * BK, left = args.K - q;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if constexpr (kSplit) {
        u32x4 high, low;
        split_chunk<T>(__builtin_bit_cast(f32x4, load_chunk<F32>(x, k + c * V, left)),
                       __builtin_bit_cast(f32x4, load_chunk<F32>(x, k + c * V + 4, left)), high, low);
        const u32x4 wv = load_chunk<T>(w[0], k + c * V, left);
        acc[0] = mfma_chunk<T>(wv, high, acc[0]);
        acc[1] = mfma_chunk<T>(wv, low, acc[1]);
      } else {
        const u32x4 xv = load_chunk<T>(x, k + c * V, left);
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g] = mfma_chunk<T>(load_chunk<T>(w[g], k + c * V, left), xv, acc[g]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < A; ++g) sums[wave][g][lane] = acc[g];
  __syncthreads();
  if (wave != 0) return;
  const int m = lane % 16, n = n0 + lane / 16 * 4;
  f32x4 total[A] = {};
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int g = 0; g < A; ++g) total[g] += sums[i][g][lane];
  if (m >= args.M) return;
  float a[4] = {total[0][0], total[0][1], total[0][2], total[0][3]};
  if constexpr (kSplit) {
#pragma unroll
    for (int e = 0; e < 4; ++e)  // of an infinite weight the rest, zero or of either sign, says nothing
      if (__builtin_isfinite(a[e])) a[e] += total[1][e];
  }
  if constexpr (GATE) {
    const float b[4] = {total[1][0], total[1][1], total[1][2], total[1][3]};
    float h[4], none[4];
    activate<false>(a, args.act, h, none);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] *= b[e];
    store4<F32>(static_cast<float*>(args.out) + int64_t(m) * args.ldo, n, args.N, h);
    if (args.g) {
      store4<F32>(args.g + int64_t(m) * args.ldg, n, args.N, a);
      store4<F32>(args.u + int64_t(m) * args.ldg, n, args.N, b);
    }
  } else {
    store4<T>(static_cast<S*>(args.out) + int64_t(m) * args.ldo, n, args.N, a);
  }
}

// A copy of an operand's rows with zeros up to the stride ldt, a multiple of a chunk: for rows that do not start on words (a
// row that starts in the middle of one would have its last element in a word that the hardware's check of a buffer's end
// refuses) and for rows that end inside a chunk.
template <typename S>
__global__ __launch_bounds__(kThreads) void k_ffn_pack(const S* from, int64_t ld, S* to, int64_t ldt, int64_t rows, int32_t cols) {
  constexpr int V = 16 / int(sizeof(S));
  typedef S vec __attribute__((ext_vector_type(V), aligned(sizeof(S))));
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int32_t c = int32_t(threadIdx.x) * V; c < ldt; c += kThreads * V) {
      const CAME8_GLOBAL S* p = gbl(from) + r * ld + c;
      vec x;
      if (c + V <= cols) {
        x = *(const CAME8_GLOBAL vec*)p;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = c + e < cols ? p[e] : S(0);
      }
      *(CAME8_GLOBAL vec*)(gbl(to) + r * ldt + c) = x;
    }
}

}  // namespace came8
