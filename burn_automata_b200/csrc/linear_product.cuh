// linear_product.cuh -- the tensor-core product of the linear operator and its
// backward pass: C = A B^T over tiles of 128 rows, with the layer's epilogue.
//
// A block has one tile at a time and walks them in a grid-stride loop.  Its
// warps have roles: producers fill a ring of operand stages (64 values of k),
// one thread issues the tensor-core products into one of two accumulator
// buffers in TMEM, and eight epilogue warps read the other one, so a tile's
// epilogue runs under the next tile's products.
//
// Operands come in two ways.  16-bit operands whose rows start on 16 bytes are
// copied by TMA into the 128-byte swizzle.  Everything else (f32, odd widths)
// goes through eight loader warps that read rows with plain loads of whatever
// alignment they have and write the same swizzled tiles.
//
// f32 values are split into three bf16 parts, x = x0 + x1 + x2 exactly but for
// 2^-24 |x| (2^-134 for the smallest), and six of the nine part products are
// summed in f32:
//   x w ~ x0 w0 + (x0 w1 + x1 w0 + x1 w1 + x0 w2 + x2 w0).
// The first two parts are cut and not rounded, so the rest, x1 w2 + x2 w1, has the
// product's sign: up to 2^-21 |x w|, 0.7 x 2^-24 in the mean over normal values.
// Sums of 256 to 4,096 terms of one sign come out 6e-8 low, 2.5e-7 off at most (the
// library's f32 product 1e-6).  Rounded parts cost the loader warps 5 to 15 %
// (8192 x 4096 x 4096 1.55 ms, 1.48).
// The tensor core truncates as it accumulates, so the leading products and the
// five small ones have accumulators of their own, and every 256 values of k the
// epilogue warps move both into rounded f32 sums in registers.
// An infinite or NaN value is whole in its first part
// and its rest is NaN: where the leading sum is not finite it is the result, and
// the small one is left out.  (An infinity times an f32 below 2^-133, whose
// first part is zero, gives NaN.)  Such values cost no time: a backward pass of
// 16384 x 1024 x 1024 takes 434 us, and 425 with every gradient NaN.
//
// 16-bit operands sum all of a tile's k in TMEM up to 128 blocks of k, 512
// accumulating steps.  Terms of one sign lose 1.1e-7 of their sum at each
// (measured with f16 over 65,536 to 1,048,576 values of k), so 512 steps stay
// below 2^-14, an eighth of f16's rounding.  A longer k moves its sums every
// 128 blocks to registers as f32 operands do: unmoved, a weight gradient over
// 1,048,576 rows came out 0.7 % low.
//
// Measured on one B200.  bf16 8192 x 4096 x 4096 in pairs' tiles: 170 us, the
// library's product 180; with the tanh gelu and a residual 185, and 220 back to
// back, where the power limit lowers the clock (tensor pipe 81 % busy).  With
// little k the epilogue and DRAM bound: 1048576 x 64 x 128 with relu and the
// pre-activation kept takes 116 us, 5.8 TB/s.  f32 8192 x 4096 x 4096 takes 1.5
// ms, 180 TFLOP/s (the library's f32 product 54): a k block's 24 products of 128
// columns and the loader warps' splits of its values take about as long.
//
// The issuing warp runs whole and one lane's products are let through: with
// loop state and descriptors in uniform registers a k block costs it few
// instructions.  A branch to one thread instead took 222 us for the first shape.
#pragma once

#include "layers.h"
#include "tcgen05.cuh"

namespace npa {
namespace linear_tc {

constexpr int kBM = 128;                 // rows of a tile: the tensor core's M
constexpr int kBK = 64;                  // k values per stage: one 128-byte swizzle row
constexpr int kEpilogueWarps = 8;        // two per 32 TMEM lanes
constexpr int kLoaderWarps = 8;
constexpr int kChunkBlocks = 4;          // k blocks between f32 moves out of TMEM
constexpr int kLongBlocks = 128;         // the same for 16-bit operands
constexpr int kSmemLimit = 227 * 1024;

// One operand: value (i, k) at i * ld + k, or at k * ld + i when MN-major.
struct Operand {
  const void* p;
  int64_t ld;
  int mn_major;
  int rows, width;  // as it lies in memory; the width may count zeros past k or m
};

struct Product {
  Operand a, b;  // [m][k] and [n][k]
  int m, n, k;
  int m_tiles, n_tiles, splits;
  int k_blocks, split_blocks;  // 64-value blocks in all and per split
  uint32_t idesc;
  int a_vec, b_vec;  // values per plain load (loader warps)
  int whole_chunks;  // both operands' chunks are all there or not at all, and aligned
  const void* bias;
  const void* residual;
  int64_t residual_stride;
  void* y;
  int64_t y_stride;
  void* z;
  int64_t z_stride;
  float* partials;  // split: [splits][layer_rows][partial_pitch], else null
  int long_k;  // 16-bit operands: more than kLongBlocks in a split
  int64_t layer_rows, partial_pitch;
  int act;
  int y_tma, z_tma, residual_vec;
};

__device__ unsigned long long g_timeouts = 0;  // bounded waits that gave up

// PAIR: two blocks (a cluster) have a tile of 256 rows, each its 128 rows of A
// and half of B's rows: a block then fetches 32 KB for 512 cycles of products
// instead of 48 KB, within what L2 delivers.
template <class T, bool LOADER, int BN, bool PAIR>
struct Config {
  static constexpr int kTileRows = PAIR ? 2 * kBM : kBM;
  static constexpr int kBRows = PAIR ? BN / 2 : BN;  // rows of B in one block
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  static constexpr int kABytes = kBM * 128, kBBytes = kBRows * 128;
  static constexpr int kStageBytes = kParts * (kABytes + kBBytes);
  // Two staging buffers to an epilogue warp where they fit: the next group is
  // written while TMA reads the last.
  static constexpr int kOutBuffers = (BN == 256 && !PAIR) || kParts == 3 ? 1 : 2;
  static constexpr int kOutBytes = kEpilogueWarps * kOutBuffers * 4096;
  static constexpr int kStagesFit = (kSmemLimit - kOutBytes - 2048 - 256) / kStageBytes;
  static constexpr int kStages = kStagesFit > 6 ? 6 : kStagesFit;
  static constexpr int kBufferColumns = BN * (kParts == 3 ? 2 : 1);
  static constexpr int kTmemColumns = 2 * kBufferColumns;
  // epilogue warps, a warpgroup with the issuing and the TMA warp, loader warps
  static constexpr int kThreads = 32 * (kEpilogueWarps + 4 + (LOADER ? kLoaderWarps : 0));
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kOutBytes + 2048 + 256;
  static_assert(kStages >= 2 && kTmemColumns <= 512, "tile does not fit");
};

// act(z) and act'(z).  NaN stays NaN.  FAST (16-bit storage): exponentials and
// reciprocals by the approximate instructions, without the library's handling of
// subnormal values, and erf by a short formula: relative errors below 1e-4, a
// fifth of f16's unit, in the tails too.  f32 storage takes the library's exp.
template <bool FAST>
__device__ __forceinline__ float exponential(float x) {
  if (!FAST) return expf(x);
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
// 1 / (1 + e^-z).  Where e^-z overflows both forms give 0.
__device__ __forceinline__ float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The same with one Newton step: within an ulp or two, at a fifth of the
// division's instructions, for x from 2^-126 to 2^126; 0 from there to 1e38.
__device__ __forceinline__ float near_reciprocal(float x) {
  const float r = fast_reciprocal(x);
  return fmaf(r, fmaf(-x, r, 1.0f), r);
}
template <bool FAST>
__device__ __forceinline__ float logistic(float z) {
  if (FAST) return fast_reciprocal(1.0f + exponential<true>(-z));
  return near_reciprocal(fminf(1.0f + expf(-z), 1e38f));  // 1e38 stands for all beyond
}
// The normal distribution function at z, with e = exp(-z^2 / 2):
// Phi(-a) = e^(-a^2 / 2) t Q(t), t = 1 / (1 + 0.2925 a), Q of degree five fitted to
// erfcx for an error below 1e-4 of Phi and below 1e-7 (least largest of the two
// over a from 0 to 14; 2.4e-7 and 7e-5 as evaluated).  An eighth of f16's unit
// down to where Phi leaves bf16's range.
__device__ __forceinline__ float fast_normal(float z, float e) {
  const float t = fast_reciprocal(fmaf(0.2925f, fabsf(z), 1.0f));
  float q = fmaf(t, -0.0860035196f, 0.266454369f);
  q = fmaf(t, q, -0.0709493086f);
  q = fmaf(t, q, 0.167996019f);
  q = fmaf(t, q, 0.104948513f);
  q = fmaf(t, q, 0.117553867f);
  q = q * t * e;
  return z < 0.0f ? q : 1.0f - q;
}
// The same for f32: Phi(-a) = e^(-a^2 / 2) t Q(t), t = 1 / (1 + 0.35 a), Q of degree
// eight fitted to erfcx (least relative error over a from 0 to 14.5, off by 3.2e-8;
// 4e-7 as evaluated near zero).  1 + erf(z / sqrt 2) would cancel below zero:
// 6 % off at z = -5, nothing left at -5.6.
__device__ __forceinline__ float precise_normal(float z, float e) {
  const float t = near_reciprocal(fminf(fmaf(0.35f, fabsf(z), 1.0f), 1e38f));
  float q = fmaf(t, -0.0291578749f, 0.144030867f);
  q = fmaf(t, q, -0.255838898f);
  q = fmaf(t, q, 0.159319577f);
  q = fmaf(t, q, -0.0232122738f);
  q = fmaf(t, q, 0.10555247f);
  q = fmaf(t, q, 0.119821296f);
  q = fmaf(t, q, 0.139863514f);
  q = fmaf(t, q, 0.139621307f);
  q = q * t * e;
  return z < 0.0f ? q : 1.0f - q;
}
template <bool FAST>
__device__ __forceinline__ float normal(float z, float e) {
  return FAST ? fast_normal(z, e) : precise_normal(z, e);
}
template <bool FAST>
__device__ __forceinline__ float activation(int act, float z) {
  switch (act) {
    case NPA_ACTIVATION_RELU: return z < 0.0f ? 0.0f : z;
    case NPA_ACTIVATION_GELU:
      return z * normal<FAST>(z, exponential<FAST>(-0.5f * z * z));
    case NPA_ACTIVATION_GELU_TANH: {
      // (1 + tanh(u)) / 2 = logistic(2u)
      const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
      return z * logistic<FAST>(2.0f * u);
    }
    case NPA_ACTIVATION_SILU: return z * logistic<FAST>(z);
    default: return z;
  }
}
template <bool FAST>
__device__ __forceinline__ float activation_slope(int act, float z) {
  switch (act) {
    case NPA_ACTIVATION_RELU: return z <= 0.0f ? 0.0f : 1.0f;
    case NPA_ACTIVATION_GELU: {
      const float e = exponential<FAST>(-0.5f * z * z);
      return normal<FAST>(z, e) + z * 0.39894228040143268f * e;
    }
    case NPA_ACTIVATION_GELU_TANH: {
      // p = logistic(2u), and its derivative is 2 p (1 - p) u'.  p (1 - p) is zero
      // from |z| = 11 on, and its products with z one by one stay zero up to the
      // largest f32, where z^2 would be infinite
      const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
      const float p = logistic<FAST>(2.0f * u);
      const float d = p * (1.0f - p) * z;
      return p + 1.59576912160573071f * (d + d * z * (0.134145f * z));
    }
    case NPA_ACTIVATION_SILU: {
      const float s = logistic<FAST>(z);
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
}

// The activation of a thread's N values, the choice outside the loop.
template <bool FAST, int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  switch (act) {
    case NPA_ACTIVATION_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<FAST>(NPA_ACTIVATION_RELU, v[i]);
      break;
    case NPA_ACTIVATION_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<FAST>(NPA_ACTIVATION_GELU, v[i]);
      break;
    case NPA_ACTIVATION_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<FAST>(NPA_ACTIVATION_GELU_TANH, v[i]);
      break;
    case NPA_ACTIVATION_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<FAST>(NPA_ACTIVATION_SILU, v[i]);
      break;
    default: break;
  }
}
// v[i] *= act'(z[i]).
template <bool FAST, int N>
__device__ __forceinline__ void times_slope(int act, float (&v)[N], const float (&z)[N]) {
  switch (act) {
    case NPA_ACTIVATION_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= activation_slope<FAST>(NPA_ACTIVATION_RELU, z[i]);
      break;
    case NPA_ACTIVATION_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= activation_slope<FAST>(NPA_ACTIVATION_GELU, z[i]);
      break;
    case NPA_ACTIVATION_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= activation_slope<FAST>(NPA_ACTIVATION_GELU_TANH, z[i]);
      break;
    case NPA_ACTIVATION_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= activation_slope<FAST>(NPA_ACTIVATION_SILU, z[i]);
      break;
    default: break;
  }
}

// The shared-memory address of 16-byte chunk c of row r in a tile of 128-byte
// rows: TMA's 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
  return uint32_t(r * 128 + ((c ^ (r & 7)) << 4));
}
__device__ __forceinline__ void store_shared16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ uint4 load_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// A position in a ring of N slots and the parity of its current phase.
template <int N>
struct Cursor {
  uint32_t slot = 0, parity = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == N) {
      slot = 0;
      parity ^= 1;
    }
  }
};

// ---- loader warps ----
// Sixteen bytes of a line: eight 16-bit values or four f32.  A warp then reads
// whole lines with each instruction: nothing is left for a second access to find
// in the L1, which beside these stages has room for less than the loads in flight.
template <class T>
struct alignas(16) Chunk {
  static constexpr int kValues = 16 / int(sizeof(T));
  T v[kValues];
};
// Zero past `valid`; `vec` values at a time where all are there.
template <class T>
__device__ __forceinline__ void load_chunk(const T* p, int valid, int vec, Chunk<T>& c) {
  constexpr int kMost = Chunk<T>::kValues;
  if (valid >= kMost) {
    if (vec == kMost) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      c = *reinterpret_cast<const Chunk<T>*>(&u);
      return;
    }
    if (vec >= 2) {
#pragma unroll
      for (int i = 0; i < kMost; i += 2)
        *reinterpret_cast<Pack<T, 2>*>(c.v + i) = *reinterpret_cast<const Pack<T, 2>*>(p + i);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kMost; ++i) c.v[i] = i < valid ? p[i] : T(0.0f);
}
__device__ __forceinline__ uint32_t high_halves(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
// Two f32 to bf16 towards zero, the low half first: no finite value becomes
// infinite, and every NaN stays one (its payload's upper half may be zero).
__device__ __forceinline__ uint32_t pack2_down(float lo, float hi) {
  uint32_t r;
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float truncated(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}
__device__ __forceinline__ void store_shared8(uint32_t addr, uint32_t lo, uint32_t hi) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(addr), "r"(lo), "r"(hi) : "memory");
}
// Where chunk `c` of line `line` goes in a tile of 128-byte lines.
template <class T>
__device__ __forceinline__ uint32_t chunk_place(int line, int c) {
  return sizeof(T) == 4 ? swizzled(line, c >> 1) + (c & 1) * 8 : swizzled(line, c);
}
// Writes the chunk's part(s) at `at`, parts `part_bytes` apart.
template <class T>
__device__ __forceinline__ void store_chunk(uint32_t at, uint32_t part_bytes, const Chunk<T>& c) {
  if constexpr (sizeof(T) == 2) {
    store_shared16(at, *reinterpret_cast<const uint4*>(c.v));
  } else {
    const F2 minus = f2(-1.0f, -1.0f);
    float r1[4], r2[4];
    uint32_t first[2];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      first[i / 2] = pack2_down(c.v[i], c.v[i + 1]);
      const float2 f = unpack2<__nv_bfloat16>(first[i / 2]);
      const float2 a = values(fma2(f2(f.x, f.y), minus, f2(c.v[i], c.v[i + 1])));
      r1[i] = a.x;
      r1[i + 1] = a.y;
      const float2 b = values(fma2(f2(truncated(a.x), truncated(a.y)), minus, f2(a.x, a.y)));
      r2[i] = b.x;
      r2[i + 1] = b.y;
    }
    store_shared8(at, first[0], first[1]);
    store_shared8(at + part_bytes, high_halves(r1[0], r1[1]), high_halves(r1[2], r1[3]));
    store_shared8(at + 2 * part_bytes, pack2<__nv_bfloat16>(r2[0], r2[1]),
                  pack2<__nv_bfloat16>(r2[2], r2[3]));
  }
}
// A loader thread's place in an operand's tiles.  A tile has lines of 64 values,
// over k for K-major operands and over m (or n) for MN-major ones; the thread
// has the same chunk of every kLines-th line.
template <class T>
struct TileReader {
  static constexpr int kLineChunks = 64 / Chunk<T>::kValues;
  static constexpr int kLines = kLoaderWarps * 32 / kLineChunks;  // at once
  static constexpr int kPasses = 64 / kLines;                     // over 64 lines
  const char* origin;    // the thread's chunk in its first line of the block
  int64_t pass_bytes;    // from one of its lines to the next
  int64_t across_bytes;  // from one run of kPasses passes to the next
  int outer, inner;      // of the first line: its row, and the values' place in it

  __device__ __forceinline__ void enter(const Operand& o, int o0, int k0, int tid) {
    const int line = tid / kLineChunks, e = tid % kLineChunks * Chunk<T>::kValues;
    outer = (o.mn_major ? k0 : o0) + line;
    inner = (o.mn_major ? o0 : k0) + e;
    origin = static_cast<const char*>(o.p) + (outer * o.ld + inner) * int64_t(sizeof(T));
    pass_bytes = kLines * o.ld * int64_t(sizeof(T));
    across_bytes = o.mn_major ? 64 * int64_t(sizeof(T)) : kPasses * pass_bytes;
  }
  __device__ __forceinline__ void next_block(const Operand& o) {
    if (o.mn_major) {
      origin += kPasses * pass_bytes;
      outer += kBK;
    } else {
      origin += kBK * int(sizeof(T));
      inner += kBK;
    }
  }
  // Pass i: lines kLines i on (MN-major: after 64 lines of k the next 64 values).
  __device__ __forceinline__ const T* at(int i) const {
    return reinterpret_cast<const T*>(origin + i % kPasses * pass_bytes + i / kPasses * across_bytes);
  }
  // vec: values per load that the operand allows.
  __device__ __forceinline__ void read(const Operand& o, int vec, int i, Chunk<T>& c) const {
    const int out = outer + (o.mn_major ? i % kPasses : i) * kLines;
    const int in = inner + (o.mn_major ? i / kPasses * 64 : 0);
    const int left = out < o.rows ? o.width - in : 0;
    load_chunk<T>(left > 0 ? at(i) : reinterpret_cast<const T*>(origin), left, vec, c);
  }
  // Whether all of `passes` chunks lie inside the operand.
  __device__ __forceinline__ bool inside(const Operand& o, int passes) const {
    const int last_line = (o.mn_major ? kPasses : passes) * kLines - kLines;
    const int last_run = o.mn_major ? (passes / kPasses - 1) * 64 : 0;
    return outer + last_line < o.rows && inner + last_run < o.width;
  }
  __device__ __forceinline__ void read_inside(int i, Chunk<T>& c) const {
    *reinterpret_cast<uint4*>(c.v) = __ldg(reinterpret_cast<const uint4*>(at(i)));
  }
  // The same where every chunk lies inside or outside the operand, on 16 bytes.
  __device__ __forceinline__ void read_whole(const Operand& o, int i, Chunk<T>& c) const {
    const int out = outer + (o.mn_major ? i % kPasses : i) * kLines;
    const int in = inner + (o.mn_major ? i / kPasses * 64 : 0);
    const bool there = out < o.rows && in < o.width;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (there) u = __ldg(reinterpret_cast<const uint4*>(at(i)));
    *reinterpret_cast<uint4*>(c.v) = u;
  }
};

// ---- rows that do not start on 16 bytes ----
// `valid` (1 to N) values from any address, zero past them, N of them 16 bytes.
// 16-bit values come as the aligned words that hold them, `inside` saying that
// the value before and the value after the N also belong to the buffer; at the
// buffer's ends one by one.
template <class T>
__device__ __forceinline__ Pack<T, 16 / int(sizeof(T))> load_ragged(const T* p, int valid, bool inside) {
  constexpr int N = 16 / int(sizeof(T));
  Pack<T, N> out{};
  if constexpr (sizeof(T) == 2) {
    if (inside && valid == N) {
      const uint32_t* const w =
          reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
      uint32_t v[N / 2 + 1];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) v[i] = w[i];
      if (reinterpret_cast<uintptr_t>(p) & 2) {
        v[N / 2] = w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = __byte_perm(v[i], v[i + 1], 0x5432);
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) reinterpret_cast<uint32_t*>(out.v)[i] = v[i];
      return out;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < valid) out.v[i] = p[i];
  return out;
}

// ---- epilogue ----
// One warp's window on an output: 32 rows from row0, a 128-byte group of
// columns from col0, staged in the warp's shared-memory buffer.
template <class OUT, int NC>
__device__ __forceinline__ void stage_values(uint32_t buf, int lane, const float (&v)[NC], int first) {
  constexpr int kPer = 16 / int(sizeof(OUT));
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint4 u;
    if constexpr (sizeof(OUT) == 4) {
      u = make_uint4(__float_as_uint(v[first + c * kPer]), __float_as_uint(v[first + c * kPer + 1]),
                     __float_as_uint(v[first + c * kPer + 2]),
                     __float_as_uint(v[first + c * kPer + 3]));
    } else {
      u = make_uint4(pack2<OUT>(v[c * kPer], v[c * kPer + 1]),
                     pack2<OUT>(v[c * kPer + 2], v[c * kPer + 3]),
                     pack2<OUT>(v[c * kPer + 4], v[c * kPer + 5]),
                     pack2<OUT>(v[c * kPer + 6], v[c * kPer + 7]));
    }
    store_shared16(buf + swizzled(lane, c), u);
  }
}
// The staged group to global memory: by TMA, or row by row where the output's
// rows do not start on 16 bytes.
template <class OUT, bool RAGGED>
__device__ __forceinline__ void put_group(uint32_t buf, int lane,
                                          const CUtensorMap* map, bool tma, int x, int y_tma_row,
                                          void* out, int64_t stride, int64_t row0, int rows,
                                          int cols) {
  if (!RAGGED || tma) {
    tc::fence_async_shared();
    __syncwarp();
    if (lane == 0) {
      tc::tma_store(map, x, y_tma_row, buf);
      tc::bulk_commit();
    }
    return;
  }
  __syncwarp();
  // A lane has columns lane and lane + 32 of every row; eight rows are read from
  // shared memory before the first is written.
  constexpr int kPer = 16 / int(sizeof(OUT)), kAcross = 4 / int(sizeof(OUT));
  OUT* to = static_cast<OUT*>(out) + row0 * stride + x + lane;
  const int e = lane % kPer * int(sizeof(OUT));
  for (int r0 = 0; r0 < rows; r0 += 8) {
    uint32_t v[8][kAcross];
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int h = 0; h < kAcross; ++h) {
        const uint32_t at = buf + swizzled(r0 + r, (lane + 32 * h) / kPer) + e;
        if constexpr (sizeof(OUT) == 4)
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[r][h]) : "r"(at));
        else
          asm volatile("{ .reg .b16 t; ld.shared.b16 t, [%1]; cvt.u32.u16 %0, t; }"
                       : "=r"(v[r][h])
                       : "r"(at));
      }
#pragma unroll
    for (int r = 0; r < 8; ++r, to += stride) {
      if (r0 + r >= rows) break;
#pragma unroll
      for (int h = 0; h < kAcross; ++h)
        if (lane + 32 * h < cols) {
          if constexpr (sizeof(OUT) == 4)
            to[32 * h] = __uint_as_float(v[r][h]);
          else
            reinterpret_cast<uint16_t*>(to)[32 * h] = uint16_t(v[r][h]);
        }
    }
  }
}

// kRagged: outputs or a residual whose rows do not start on 16 bytes.  kLong: the
// same, and more than kLongBlocks of k (16-bit operands).  The common case does
// without that code: its size alone costs (1048576 x 64 x 128 bf16: 126 us with
// the ragged epilogue, 117 without).
enum Form { kWhole, kRagged, kLong };
template <class T, bool LOADER, int BN, bool PAIR, Form FORM>
__global__ void __launch_bounds__((Config<T, LOADER, BN, PAIR>::kThreads), 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_z,
               const __grid_constant__ Product p) {
  using C = Config<T, LOADER, BN, PAIR>;
  constexpr bool RAGGED = FORM != kWhole, LONG = FORM == kLong;
  constexpr int kGroup = 128 / int(sizeof(T));         // output columns staged at a time
  constexpr int kGroups = BN / kGroup;
  constexpr int kGroupsPerWarp = (kGroups + 1) / 2;
  // k blocks between moves out of TMEM, 0: none before the tile's end
  constexpr int kMoved = C::kParts == 3 ? kChunkBlocks : LONG ? kLongBlocks : 0;
  extern __shared__ char smem_raw[];
  const uint32_t raw = tc::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023) & ~1023u;  // the swizzle repeats every 1,024 bytes
  const uint32_t out_base = base + C::kStages * C::kStageBytes;
  const uint32_t bias_base = out_base + C::kOutBytes;  // 128 bytes per epilogue warp
  const uint32_t bars = bias_base + kEpilogueWarps * 128;
  const uint32_t full = bars, empty = bars + 8 * C::kStages;
  const uint32_t acc_full = empty + 8 * C::kStages, acc_empty = acc_full + 16;
  const uint32_t drain = acc_empty + 16, tmem_at = drain + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMmaWarp = kEpilogueWarps, kTmaWarp = kEpilogueWarps + 1;
  constexpr int kFirstLoader = kEpilogueWarps + 4;
  // a pair walks the tiles together
  const uint32_t rank = PAIR ? tc::cluster_rank() : 0;
  const uint32_t walker = PAIR ? blockIdx.x / 2 : blockIdx.x;
  const uint32_t walkers = PAIR ? gridDim.x / 2 : gridDim.x;
  const uint32_t layer = uint32_t(p.m_tiles) * p.n_tiles;  // the host keeps tiles below 2^31
  const uint32_t tiles = layer * p.splits;

  let_next_launch();
  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int s = 0; s < C::kStages; ++s) {
        tc::bar_init(full + 8 * s, LOADER ? kLoaderWarps : 1);
        tc::bar_init(empty + 8 * s, 1);
      }
      for (int b = 0; b < 2; ++b) {
        tc::bar_init(acc_full + 8 * b, 1);
        tc::bar_init(acc_empty + 8 * b, kEpilogueWarps * (PAIR ? 2 : 1));
      }
      tc::bar_init(drain, 1);
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    tc::tmem_alloc<PAIR>(tmem_at, C::kTmemColumns);
    tc::fence_before();
  }
  if (warp == kTmaWarp && lane == 0) {
    if (!LOADER) {
      tc::prefetch_map(&map_a);
      tc::prefetch_map(&map_b);
    }
    if (p.y_tma) tc::prefetch_map(&map_y);
    if (p.z_tma) tc::prefetch_map(&map_z);
  }
  __syncthreads();
  if (PAIR) tc::cluster_sync();  // the other block's barriers are ready
  tc::fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(tmem) : "r"(tmem_at) : "memory");
  bool ok = true;
  wait_for_previous();

  // The loader kernel's 640 threads start with 96 registers each; its control
  // warpgroup leaves some to the others: 56 + 2 x 96 + 2 x 112 = 472 of the
  // launch's 480 per thread of each warpgroup.  The TMA kernels' 384 threads start
  // with 168; where sums stay in registers over a long k the two epilogue
  // warpgroups get 224 each and the control warpgroup keeps 56: all 504.
  if (warp > kMmaWarp) {
    // ---- producers ----
    if (!LOADER) {
      if constexpr (LONG) tc::registers_down<56>();
      if (warp == kTmaWarp && lane == 0) {
        Cursor<C::kStages> at;
        uint32_t issued = 0;
        const uint32_t first_full = PAIR ? tc::in_first_block(full) : full;
        for (uint32_t t = walker; t < tiles && ok; t += walkers) {
          const int split = p.splits > 1 ? int(t / layer) : 0, in = int(t - split * layer);
          const int m0 = in / p.n_tiles * C::kTileRows + int(rank) * kBM;
          const int n0 = in % p.n_tiles * BN + int(rank) * C::kBRows;
          const int kb = split * p.split_blocks;
          const int ke = min(p.k_blocks, kb + p.split_blocks);
          for (int kt = kb; kt < ke; ++kt, at.advance()) {
            const uint32_t s = at.slot;
            ok = tc::bar_wait(empty + 8 * s, at.parity ^ 1);
            if (!ok) break;
            if (issued < C::kStages) ++issued;
            const uint32_t a = base + s * C::kStageBytes, b = a + C::kABytes;
            const uint32_t bar = PAIR ? first_full + 8 * s : full + 8 * s;
            if (rank == 0)
              tc::bar_expect(full + 8 * s, (C::kABytes + C::kBBytes) * (PAIR ? 2 : 1));
            auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
              if (PAIR)
                tc::tma_load_pair(dst, map, x, y, bar);
              else
                tc::tma_load(dst, map, x, y, bar);
            };
            if (p.a.mn_major) {
#pragma unroll
              for (int i = 0; i < kBM / 64; ++i) load(a + i * 8192, &map_a, m0 + i * 64, kt * kBK);
            } else {
              load(a, &map_a, kt * kBK, m0);
            }
            if (p.b.mn_major) {
#pragma unroll
              for (int i = 0; i < C::kBRows / 64; ++i)
                load(b + i * 8192, &map_b, n0 + i * 64, kt * kBK);
            } else {
              load(b, &map_b, kt * kBK, n0);
            }
          }
        }
        // copies in flight must land before the block may leave (the second block
        // of a pair has no barrier of its own for them: the wait that gave up was
        // a million times their latency)
        if (!ok && rank == 0) {
          for (uint32_t j = 0; j < issued; ++j) {  // backwards from the slot not filled
            const uint32_t slot = (at.slot + C::kStages - 1 - j) % C::kStages;
            tc::bar_wait(full + 8 * slot, slot < at.slot ? at.parity : at.parity ^ 1);
          }
        }
      }
    } else {
      if (warp < kFirstLoader) {
        tc::registers_down<56>();
      } else {
        tc::registers_up<112>();
        // A thread has up to 32 registers of A's tile and of B's, loaded a stage
        // ahead of their use.
        const int tid = threadIdx.x - kFirstLoader * 32;
        using Reader = TileReader<T>;
        constexpr int kAChunks = kBM / Reader::kLines, kBChunks = BN / Reader::kLines;
        Cursor<C::kStages> at;
        Chunk<T> ca[kAChunks], cb[kBChunks];
        Reader ra, rb;
        uint32_t t = walker;
        int blocks_left = 0;
        auto enter_tile = [&]() {
          const int split = p.splits > 1 ? int(t / layer) : 0, in = int(t - split * layer);
          const int m0 = in / p.n_tiles * kBM, n0 = in % p.n_tiles * BN;
          const int kb = split * p.split_blocks;
          blocks_left = min(p.k_blocks, kb + p.split_blocks) - kb;
          ra.enter(p.a, m0, kb * kBK, tid);
          rb.enter(p.b, n0, kb * kBK, tid);
        };
        auto read_all = [&]() {
#pragma unroll
          for (int i = 0; i < kAChunks; ++i) ra.read(p.a, p.a_vec, i, ca[i]);
#pragma unroll
          for (int i = 0; i < kBChunks; ++i) rb.read(p.b, p.b_vec, i, cb[i]);
        };
        if (t < tiles) {
          enter_tile();
          if (p.whole_chunks) {
#pragma unroll
            for (int i = 0; i < kAChunks; ++i) ra.read_whole(p.a, i, ca[i]);
#pragma unroll
            for (int i = 0; i < kBChunks; ++i) rb.read_whole(p.b, i, cb[i]);
          } else {
            read_all();
          }
        }
        for (; t < tiles; at.advance()) {
          ok = tc::bar_wait(empty + 8 * at.slot, at.parity ^ 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (--blocks_left == 0) {
            t += walkers;
            if (t < tiles) enter_tile();
          } else {
            ra.next_block(p.a);
            rb.next_block(p.b);
          }
          const bool more = t < tiles;
          const uint32_t a = base + at.slot * C::kStageBytes +
                             chunk_place<T>(tid / Reader::kLineChunks, tid % Reader::kLineChunks);
          const uint32_t b = a + C::kParts * C::kABytes;
          // Straight-line code, whose splits overlap: a register chunk is asked for
          // again, for the next stage, as soon as it has been written.  Inside the
          // operands without predicates (8192 x 4096 x 4096 f32: 1.51 ms, 1.81 with).
          if (p.whole_chunks &&
              __all_sync(0xffffffffu, more && ra.inside(p.a, kAChunks) && rb.inside(p.b, kBChunks))) {
#pragma unroll
            for (int i = 0; i < kAChunks; ++i) {
              store_chunk<T>(a + i * Reader::kLines * 128, C::kABytes, ca[i]);
              ra.read_inside(i, ca[i]);
            }
#pragma unroll
            for (int i = 0; i < kBChunks; ++i) {
              store_chunk<T>(b + i * Reader::kLines * 128, C::kBBytes, cb[i]);
              rb.read_inside(i, cb[i]);
            }
          } else if (p.whole_chunks) {
#pragma unroll
            for (int i = 0; i < kAChunks; ++i) {
              store_chunk<T>(a + i * Reader::kLines * 128, C::kABytes, ca[i]);
              if (more) ra.read_whole(p.a, i, ca[i]);
            }
#pragma unroll
            for (int i = 0; i < kBChunks; ++i) {
              store_chunk<T>(b + i * Reader::kLines * 128, C::kBBytes, cb[i]);
              if (more) rb.read_whole(p.b, i, cb[i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < kAChunks; ++i)
              store_chunk<T>(a + i * Reader::kLines * 128, C::kABytes, ca[i]);
#pragma unroll
            for (int i = 0; i < kBChunks; ++i)
              store_chunk<T>(b + i * Reader::kLines * 128, C::kBBytes, cb[i]);
          }
          // no proxy fence here: it would wait for the loads in flight.  The thread
          // that issues the products has one, after this barrier.
          __syncwarp();
          if (lane == 0) tc::bar_arrive(full + 8 * at.slot);
          if (more && !p.whole_chunks) read_all();
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ---- the warp that issues the products (the pair's first block's) ----
    if constexpr (LOADER || LONG) tc::registers_down<56>();
    if (rank == 0) {
      // One lane issues everything, so what lies between two blocks of k counts:
      // the warp runs whole, cursors step by one and descriptors by additions.
      const uint32_t issue = tc::elected();
      Cursor<C::kStages> at;
      Cursor<2> acc;
      const uint32_t a_step = (p.a.mn_major ? 2048 : 32) >> 4, b_step = (p.b.mn_major ? 2048 : 32) >> 4;
      const uint64_t a0 = tc::operand_desc(base, p.a.mn_major, 8192);
      const uint64_t b0 = tc::operand_desc(base + C::kParts * C::kABytes, p.b.mn_major, 8192);
      for (uint32_t t = walker; t < tiles && ok; t += walkers) {
        const int split = p.splits > 1 ? int(t / layer) : 0;
        const int kb = split * p.split_blocks;
        const int blocks = min(p.k_blocks, kb + p.split_blocks) - kb;
        // a last block may end early: steps past k's end are left out
        const int last_steps = min(kBK / 16, (p.k - (kb + blocks - 1) * kBK + 15) / 16);
        uint32_t d = 0;
        int in_chunk = 0;
        for (int kt = 0; kt < blocks; ++kt, at.advance()) {
          if (in_chunk == 0) {
            ok = __all_sync(0xffffffffu, tc::bar_wait<PAIR>(acc_empty + 8 * acc.slot, acc.parity ^ 1));
            if (!ok) break;
            d = tmem + acc.slot * C::kBufferColumns;
          }
          ok = __all_sync(0xffffffffu, tc::bar_wait(full + 8 * at.slot, at.parity));
          if (!ok) break;
          if (LOADER) tc::fence_async_shared();  // the loaders' writes, ordered by the barrier
          tc::fence_after();
          const uint64_t a = a0 + at.slot * (C::kStageBytes >> 4), b = b0 + at.slot * (C::kStageBytes >> 4);
          auto products = [&](int step) {
            const bool more = step > 0 || in_chunk > 0;
            const uint64_t as = a + step * a_step, bs = b + step * b_step;
            tc::mma_f16<PAIR>(d, as, bs, p.idesc, more, issue);
            if constexpr (C::kParts == 3) {
              constexpr int kA[5] = {0, 1, 1, 0, 2}, kB[5] = {1, 0, 1, 2, 0};
#pragma unroll
              for (int j = 0; j < 5; ++j)
                tc::mma_f16<PAIR>(d + BN, as + kA[j] * (C::kABytes >> 4), bs + kB[j] * (C::kBBytes >> 4),
                                  p.idesc, more || j > 0, issue);
            }
          };
          if (kt + 1 < blocks || last_steps == kBK / 16) {
#pragma unroll
            for (int step = 0; step < kBK / 16; ++step) products(step);
          } else {
            for (int step = 0; step < last_steps; ++step) products(step);
          }
          tc::mma_commit<PAIR>(empty + 8 * at.slot, issue);
          ++in_chunk;
          if (kt + 1 == blocks || (kMoved > 0 && in_chunk == kMoved)) {
            tc::mma_commit<PAIR>(acc_full + 8 * acc.slot, issue);
            acc.advance();
            in_chunk = 0;
          }
        }
      }
      if (!ok) {  // products in flight must end before TMEM is freed
        tc::mma_commit<PAIR>(drain, issue);
        tc::bar_wait(drain, 0);
      }
    }
  } else {
    // ---- epilogue warps: 32 rows each, every other group of columns ----
    if constexpr (LONG && !LOADER) tc::registers_up<224>();
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t bufs = out_base + warp * C::kOutBuffers * 4096;
    const uint32_t first_acc_empty = PAIR ? tc::in_first_block(acc_empty) : acc_empty;
    uint32_t turn = 0;
    Cursor<2> acc;
    // the next staging buffer, free of its last copy
    auto next_buffer = [&]() -> uint32_t {
      if (lane == 0) tc::bulk_wait_read<C::kOutBuffers - 1>();
      __syncwarp();
      const uint32_t b = bufs + (turn % C::kOutBuffers) * 4096;
      ++turn;
      return b;
    };
    auto release_accumulators = [&](uint32_t buf) {
      tc::fence_before();
      __syncwarp();
      if (lane != 0) return;
      if (PAIR)
        tc::bar_arrive_cluster(first_acc_empty + 8 * buf);
      else
        tc::bar_arrive(acc_empty + 8 * buf);
    };
    auto pointer = [&](uint32_t b) -> char* { return smem_raw + (b - raw); };
    T* const bias_row = reinterpret_cast<T*>(pointer(bias_base + warp * 128));
    // The bias of the next group, a value or two per lane, loaded a group ahead in
    // the TMA kernels: there is hardly any L1 beside the stages, so even what all
    // rows share comes from L2 each time, 600 cycles away and more.  The loader
    // kernels read it in place: their epilogue warps have no registers for it
    // (858187 x 64 x 48 f32: 102 us, 118 ahead).
    T bias_values[kGroup / 32];
    auto prefetch_bias = [&](uint32_t tile, int gi) {
      if (!p.bias || p.partials || tile >= tiles) return;
      const int in = int(p.splits > 1 ? tile % layer : tile);
      const int col0 = in % p.n_tiles * BN + (half + 2 * gi) * kGroup;
#pragma unroll
      for (int h = 0; h < kGroup / 32; ++h) {
        const int c = col0 + lane + 32 * h;
        bias_values[h] = c < p.n ? static_cast<const T*>(p.bias)[c] : T(0.0f);
      }
    };
    if (!LOADER) prefetch_bias(walker, 0);
    for (uint32_t t = walker; t < tiles && ok; t += walkers) {
      const int split = p.splits > 1 ? int(t / layer) : 0, in = int(t - split * layer);
      const int m_tile = in / p.n_tiles;
      const int64_t row0 = int64_t(m_tile) * C::kTileRows + rank * kBM + quarter * 32;
      const int n0 = in % p.n_tiles * BN;
      const int64_t rows_left = int64_t(p.m) - row0;
      const int rows = rows_left >= 32 ? 32 : rows_left > 0 ? int(rows_left) : 0;
      float sums[kMoved > 0 ? kGroupsPerWarp : 1][kGroup];
      uint32_t d = 0;
      // The TMA kernels ask for the residual before the wait for the accumulators
      // (the first group) or before they read them; the loader kernels' register
      // budget (five warps to an SM quarter) has no room for it.
      uint4 res[LOADER ? 1 : 8];
      // 16 bytes of row i * 4 + lane / 8; or, where rows do not start on 16 bytes,
      // words i * 4 .. + 3 of the lane's columns lane and lane + 32 of half the
      // rows: an access has to take all of what it touches
      auto residual_at = [&](int col0, int cols, int i, int half_rows) -> uint4 {
        const bool res_vec = !RAGGED || (p.residual_vec && cols * int(sizeof(T)) % 16 == 0);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (res_vec) {
          const int rr = i * 4 + (lane >> 3), c = (lane & 7) * (16 / int(sizeof(T)));
          if (rr < rows && c < cols)
            u = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) +
                                                (row0 + rr) * p.residual_stride + col0 + c);
          return u;
        }
        constexpr int kAcross = kGroup / 32;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int rr = half_rows + (i * 4 + q) / kAcross, c = lane + 32 * ((i * 4 + q) % kAcross);
          w[q] = 0;
          if (rr < rows && c < cols) {
            const T* const r = static_cast<const T*>(p.residual) + (row0 + rr) * p.residual_stride + col0 + c;
            if constexpr (sizeof(T) == 4)
              w[q] = *reinterpret_cast<const uint32_t*>(r);
            else
              w[q] = *reinterpret_cast<const uint16_t*>(r);
          }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
      };
      auto prefetch = [&](int gi) {
        const int g = half + 2 * gi, col0 = n0 + g * kGroup, cols = min(kGroup, p.n - col0);
        if (g >= kGroups || col0 >= p.n || rows <= 0 || p.partials) return;
        if constexpr (!LOADER) {
          if (p.residual) {
#pragma unroll
            for (int i = 0; i < 8; ++i) res[i] = residual_at(col0, cols, i, 0);
          }
        }
      };
      prefetch(0);
      if constexpr (kMoved > 0) {
        const int kb = split * p.split_blocks;
        const int blocks = min(p.k_blocks, kb + p.split_blocks) - kb;
        const int chunks = (blocks + kMoved - 1) / kMoved;
#pragma unroll
        for (int gi = 0; gi < kGroupsPerWarp; ++gi)
#pragma unroll
          for (int e = 0; e < kGroup; ++e) sums[gi][e] = 0.0f;
        for (int ch = 0; ch < chunks; ++ch, acc.advance()) {
          const uint32_t buf = acc.slot;
          ok = tc::bar_wait(acc_full + 8 * buf, acc.parity);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc::fence_after();
#pragma unroll
          for (int gi = 0; gi < kGroupsPerWarp; ++gi) {
            if constexpr (kGroups % 2 != 0)
              if (half + 2 * gi >= kGroups) continue;
            const uint32_t at = tmem + buf * C::kBufferColumns + lanes + (half + 2 * gi) * kGroup;
#pragma unroll
            for (int h = 0; h < kGroup; h += 16) {
              float part[16];
              tc::tmem_load(at + h, part);
#pragma unroll
              for (int e = 0; e < 16; ++e) sums[gi][h + e] += part[e];
              if constexpr (C::kParts == 1) continue;
              tc::tmem_load(at + BN + h, part);
              if constexpr (RAGGED) {
                // value by value: this kernel spills with the other form (backward
                // pass of 32032 x 3819 -> 13: 715 us, 672 like this)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  if (fabsf(sums[gi][h + e]) < INFINITY) sums[gi][h + e] += part[e];
              } else {
                // one vote for all (858187 x 40 x 48 silu: 131 us, 150 value by value)
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 16; ++e) odd = odd || !(fabsf(sums[gi][h + e]) < INFINITY);
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                  for (int e = 0; e < 16; ++e)
                    if (!(fabsf(sums[gi][h + e]) < INFINITY)) part[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) sums[gi][h + e] += part[e];
              }
            }
          }
          release_accumulators(buf);
        }
        if (!ok) break;
      } else {
        const uint32_t buf = acc.slot;
        ok = tc::bar_wait(acc_full + 8 * buf, acc.parity);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after();
        d = tmem + buf * C::kBufferColumns + lanes;
      }
      // One group of columns; v: its sums, or room for its accumulators.
      auto finish_group = [&](int gi, float (&v)[kGroup]) {
        const int g = half + 2 * gi;
        const int col0 = n0 + g * kGroup;
        const bool last = gi + 1 == kGroupsPerWarp;
        const bool mine = g < kGroups && col0 < p.n && rows > 0;
        const int cols = min(kGroup, p.n - col0);
        const bool res_vec = !RAGGED || (p.residual_vec && cols * int(sizeof(T)) % 16 == 0);
        auto read_residual = [&](int i, int half_rows) { return residual_at(col0, cols, i, half_rows); };
        auto stage_residual = [&](uint32_t b, int i, int half_rows, uint4 u) {
          if (res_vec) {
            store_shared16(b + swizzled(i * 4 + (lane >> 3), lane & 7), u);
            return;
          }
          constexpr int kAcross = kGroup / 32, kPer = 16 / int(sizeof(T));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int rr = half_rows + (i * 4 + q) / kAcross, c = lane + 32 * ((i * 4 + q) % kAcross);
            const uint32_t at = b + swizzled(rr, c / kPer) + c % kPer * int(sizeof(T));
            if constexpr (sizeof(T) == 4)
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(w[q]) : "memory");
            else
              asm volatile("{ .reg .b16 t; cvt.u16.u32 t, %1; st.shared.b16 [%0], t; }" ::"r"(at), "r"(w[q])
                           : "memory");
          }
        };
        if (gi > 0) prefetch(gi);
        if (LOADER) prefetch_bias(t, gi);
        if constexpr (kMoved == 0) {
          if (mine) tc::tmem_load(d + g * kGroup, v);
          if (last) {
            release_accumulators(acc.slot);
            acc.advance();
          }
        }
        if (!mine) {
          if (!LOADER && last) prefetch_bias(t + walkers, 0);
          return;
        }
        if (p.partials) {
          const int64_t prow = split * p.layer_rows + row0;
#pragma unroll
          for (int h = 0; h < kGroup / 32; ++h) {
            if (h * 32 >= cols) break;
            const uint32_t b = next_buffer();
            stage_values<float>(b, lane, v, h * 32);
            put_group<float, false>(b, lane, &map_y, true, col0 + h * 32, int(prow), nullptr,
                             0, 0, 0, 0);
          }
          return;
        }
        if (p.bias) {
          // through shared memory to all lanes: each has a row of its own
          __syncwarp();
#pragma unroll
          for (int h = 0; h < kGroup / 32; ++h) bias_row[lane + 32 * h] = bias_values[h];
          __syncwarp();
          if (!LOADER) prefetch_bias(last ? t + walkers : t, last ? 0 : gi + 1);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            constexpr int kPer = 16 / int(sizeof(T));
            const Pack<T, kPer> b = reinterpret_cast<const Pack<T, kPer>*>(bias_row)[c];
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[c * kPer + j] += to_f32(b.v[j]);
          }
        }
        if (p.z) {
          const uint32_t b = next_buffer();
          stage_values<T>(b, lane, v, 0);
          put_group<T, RAGGED>(b, lane, &map_z, p.z_tma, col0, int(row0), p.z, p.z_stride,
                       row0, rows, cols);
        }
        activate<sizeof(T) == 2>(p.act, v);
        const uint32_t b = next_buffer();
        if (p.residual) {
          if constexpr (LOADER) {
            for (int i = 0; i < 8; ++i) stage_residual(b, i, 0, read_residual(i, 0));
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) stage_residual(b, i, 0, res[i]);
          }
          // 32 single values per lane are all of 32 f32 columns, and half of the
          // rows of 64 columns
          if (RAGGED && kGroup == 64 && !res_vec) {
            constexpr int kAt = 16;
            if constexpr (LOADER) {
              for (int i = 0; i < 8; ++i) stage_residual(b, i, kAt, read_residual(i, kAt));
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) res[i] = read_residual(i, kAt);
#pragma unroll
              for (int i = 0; i < 8; ++i) stage_residual(b, i, kAt, res[i]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint4 u = load_shared16(b + swizzled(lane, c));
            if constexpr (sizeof(T) == 4) {
              v[c * 4] += __uint_as_float(u.x);
              v[c * 4 + 1] += __uint_as_float(u.y);
              v[c * 4 + 2] += __uint_as_float(u.z);
              v[c * 4 + 3] += __uint_as_float(u.w);
            } else {
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 f = unpack2<T>(w[j]);
                v[c * 8 + 2 * j] += f.x;
                v[c * 8 + 2 * j + 1] += f.y;
              }
            }
          }
        }
        stage_values<T>(b, lane, v, 0);
        put_group<T, RAGGED>(b, lane, &map_y, p.y_tma, col0, int(row0), p.y, p.y_stride, row0,
                     rows, cols);
      };
#pragma unroll
      for (int gi = 0; gi < kGroupsPerWarp; ++gi) {
        if constexpr (kMoved > 0) {
          finish_group(gi, sums[gi]);
        } else {
          float v[kGroup];
          finish_group(gi, v);
        }
      }
    }
    if (lane == 0) tc::bulk_wait_all();
  }
  if (!ok && lane == 0) atomicAdd(&g_timeouts, 1ull);
  __syncthreads();
  if (PAIR) tc::cluster_sync();  // neither block leaves while the other may still reach it
  if (warp == kMmaWarp) {
    tc::fence_after();
    tc::tmem_free<PAIR>(tmem, C::kTmemColumns);
  }
}

}  // namespace linear_tc
}  // namespace npa
