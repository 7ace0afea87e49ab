// layer_norm.cu -- layer norm over rows, forward and backward.
//
// Forward, per row of n values:  mean = sum(x) / n,
// rstd = 1 / sqrt(sum((x - mean)^2) / n + eps), y = (x - mean) rstd w + b.
// The variance is summed from centred values (a second walk over the row's
// registers): sum(x^2) - n mean^2 would lose the variance of rows whose mean
// is large against their spread.
// Backward, with xhat = (x - mean) rstd and g = dy w:
//   dx = rstd (g - sum(g) / n - xhat sum(g xhat) / n) + residual gradient,
//   dw = sum over rows of dy xhat, db = sum over rows of dy.
// Both are bound by memory: the forward pass reads and writes each value
// once, the backward pass reads two (three with a residual) and writes one.
// A row therefore lives in registers between its reads and its writes, and
// the backward pass keeps each thread's share of dw and db in registers over
// all rows that it walks; the blocks' shares meet in a second small kernel, in
// a fixed order.
//
// How a row reaches the registers depends on how it lies in memory:
//  - rows that follow each other without gaps and are short: eight rows are a
//    whole number of 16-byte units whatever the width, so each warp has a ring
//    of eight-row tiles in shared memory, filled by bulk copies and (results in
//    place) emptied by bulk copies.  Odd widths then cost no partial accesses
//    in global memory.  layer_norm_tiles_kernel, layer_norm_backward_tiles_kernel;
//  - longer rows that start on 16 bytes: a block per row, whole rows copied
//    ahead into a ring.  layer_norm_wide_kernel, layer_norm_backward_wide_kernel;
//  - everything else (column ranges, long odd widths): plain loads.
//    layer_norm_kernel, layer_norm_backward_kernel, and walks over global memory
//    past what registers hold.
//
// Measured on one B200, beside a copy's 6.45 TB/s: forward 1048576 x 130 f32
// 178 us (6.1 TB/s; 194 on inputs that change from call to call); backward with a
// residual 1048576 x 130 bf16 209 us (5.3 TB/s, instruction issue at 70 %), 16384 x 4096 f16 83 us (4.8 TB/s); the plain
// loads of unaligned rows reach a quarter to a third (52529 x 1599 f16, odd pitch:
// forward 173 us, backward 279, with a residual 397), bound by their two-byte
// accesses.
#include <algorithm>

#include "layers.h"
#include "tcgen05.cuh"

namespace npa {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarpRowThreads = 256;  // threads per block where a warp or less has a row

// Sums over a row's threads: tpr lanes of a warp (a power of two), or the whole
// block through shared memory, whose two halves alternate so that one barrier
// per sum is enough.
struct RowSum {
  float2* buf;  // [2][16], block rows only
  int phase = 0;
};
template <bool BLOCK>
__device__ __forceinline__ void row_sum2(RowSum& rs, int tpr, float& a, float& b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (BLOCK || o < tpr) {
      a += __shfl_xor_sync(kFull, a, o);
      b += __shfl_xor_sync(kFull, b, o);
    }
  if (BLOCK) {
    float2* const s = rs.buf + rs.phase * 16;
    rs.phase ^= 1;
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
    for (int w = 0; w < warps; ++w) {
      const float2 t = s[w];
      a += t.x;
      b += t.y;
    }
  }
}
template <bool BLOCK>
__device__ __forceinline__ float row_sum(RowSum& rs, int tpr, float a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (BLOCK || o < tpr) a += __shfl_xor_sync(kFull, a, o);
  if (BLOCK) {
    float2* const s = rs.buf + rs.phase * 16;
    rs.phase ^= 1;
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) s[warp].x = a;
    __syncthreads();
    a = 0.0f;
    for (int w = 0; w < warps; ++w) a += s[w].x;
  }
  return a;
}

// ---- a thread's share of a row ----
// A thread has the accesses first, first + step, ... of VEC values, NV of them
// at most, as E values in pairs.  In global memory a row's threads lie side by
// side (first = lane, step = threads per row).  In a warp's shared-memory tile
// a thread's accesses follow each other (first = lane * NV, step = Next, known
// to the compiler): the offsets are immediates, and odd NV meet all banks.
struct Next {
  __device__ __forceinline__ constexpr operator int() const { return 1; }
};
template <int VEC, int NV>
struct Row {
  static constexpr int E = VEC * NV, kPairs = (E + 1) / 2;
  F2 v[kPairs];
};
// Past nvec (and for `active` false) the values are zero.
template <class T, int VEC, int NV, class Step>
__device__ __forceinline__ void load_row(const T* row, int first, Step step, int nvec, bool active,
                                         Row<VEC, NV>& out) {
  if constexpr (sizeof(T) == 2 && VEC >= 2) {
    // whole words: a pair of 16-bit values widens in two instructions
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = first + k * step;
      Pack<uint32_t, VEC / 2> p{};
      if (active && q < nvec) p = reinterpret_cast<const Pack<uint32_t, VEC / 2>*>(row)[q];
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const float2 t = unpack2<T>(p.v[j]);
        out.v[k * (VEC / 2) + j] = f2(t.x, t.y);
      }
    }
    return;
  }
  float f[2 * Row<VEC, NV>::kPairs];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int q = first + k * step;
    Pack<T, VEC> p{};
    if (active && q < nvec) p = reinterpret_cast<const Pack<T, VEC>*>(row)[q];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[k * VEC + j] = to_f32(p.v[j]);
  }
  if (Row<VEC, NV>::E & 1) f[Row<VEC, NV>::E] = 0.0f;
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) out.v[i] = f2(f[2 * i], f[2 * i + 1]);
}
template <class T, int VEC, int NV, class Step>
__device__ __forceinline__ void store_row(T* row, int first, Step step, int nvec, const Row<VEC, NV>& in) {
  if constexpr (sizeof(T) == 2 && VEC >= 2) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = first + k * step;
      Pack<uint32_t, VEC / 2> p;
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const float2 t = values(in.v[k * (VEC / 2) + j]);
        p.v[j] = pack2<T>(t.x, t.y);
      }
      if (q < nvec) reinterpret_cast<Pack<uint32_t, VEC / 2>*>(row)[q] = p;
    }
    return;
  }
  float f[2 * Row<VEC, NV>::kPairs];
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) {
    const float2 t = values(in.v[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int q = first + k * step;
    Pack<T, VEC> p;
#pragma unroll
    for (int j = 0; j < VEC; ++j) p.v[j] = from_f32<T>(f[k * VEC + j]);
    if (q < nvec) reinterpret_cast<Pack<T, VEC>*>(row)[q] = p;
  }
}
// A parameter vector's share: `fill` where it is absent.  Scalar loads: read
// once per thread, and only as aligned as its type.
template <class T, int VEC, int NV, class Step>
__device__ __forceinline__ void load_parameter(const void* from, int first, Step step, int nvec, float fill,
                                               Row<VEC, NV>& out) {
  float f[2 * Row<VEC, NV>::kPairs];
#pragma unroll
  for (int e = 0; e < 2 * Row<VEC, NV>::kPairs; ++e) {
    const int q = first + e / VEC * step;
    f[e] = from && e < VEC * NV && q < nvec ? to_f32(static_cast<const T*>(from)[q * VEC + e % VEC])
                                            : fill;
  }
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) out.v[i] = f2(f[2 * i], f[2 * i + 1]);
}

template <int VEC, int NV>
__device__ __forceinline__ float forward_sum(const Row<VEC, NV>& x) {
  F2 s = x.v[0];
#pragma unroll
  for (int i = 1; i < Row<VEC, NV>::kPairs; ++i) s = add2(s, x.v[i]);
  const float2 t = values(s);
  return t.x + t.y;
}
// x - mean in place (zero past nvec), and the sum of its squares.
template <int VEC, int NV, class Step>
__device__ __forceinline__ float forward_centre(Row<VEC, NV>& x, float mean, int first, Step step, int nvec) {
  F2 s = f2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) {
    const int e0 = 2 * i, e1 = 2 * i + 1;
    const bool in0 = first + e0 / VEC * step < nvec;
    const bool in1 = e1 < VEC * NV && first + e1 / VEC * step < nvec;
    x.v[i] = add2(x.v[i], f2(in0 ? -mean : 0.0f, in1 ? -mean : 0.0f));
    s = fma2(x.v[i], x.v[i], s);
  }
  const float2 t = values(s);
  return t.x + t.y;
}
template <int VEC, int NV>
__device__ __forceinline__ void forward_out(Row<VEC, NV>& x, float rstd, const Row<VEC, NV>& w,
                                            const Row<VEC, NV>& b) {
  const F2 r = f2(rstd, rstd);
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) x.v[i] = fma2(mul2(x.v[i], r), w.v[i], b.v[i]);
}

// x becomes xhat, g (dy) becomes dy w; dw, db and this thread's share of
// sum(g) and sum(g xhat) grow.  Values past the row's end are zero in dy, so
// whatever xhat holds there adds nothing that is stored.  16-bit rows take
// xhat = x rstd - mean rstd in one step: the rounded product costs 2^-24
// mean rstd, as much as the rounding of the saved mean and far below the spacing
// of the values themselves (rows of one value far from zero get that in place of
// zeros; subtracting first would cost 1048576 x 130 bf16 209 us, 191 like this);
// f32 rows subtract first.
template <class T, int VEC, int NV>
__device__ __forceinline__ void backward_sums(Row<VEC, NV>& x, Row<VEC, NV>& g, const Row<VEC, NV>& w,
                                              float mean, float rstd, bool params, Row<VEC, NV>& dw,
                                              Row<VEC, NV>& db, float& s1, float& s2) {
  const F2 r = f2(rstd, rstd);
  const float shift = sizeof(T) == 2 ? -mean * rstd : -mean;
  const F2 m = f2(shift, shift);
  F2 a = f2(0.0f, 0.0f), b = f2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) {
    x.v[i] = sizeof(T) == 2 ? fma2(x.v[i], r, m) : mul2(add2(x.v[i], m), r);
    if (params) {
      dw.v[i] = fma2(g.v[i], x.v[i], dw.v[i]);
      db.v[i] = add2(db.v[i], g.v[i]);
    }
    g.v[i] = mul2(g.v[i], w.v[i]);
    a = add2(a, g.v[i]);
    b = fma2(g.v[i], x.v[i], b);
  }
  const float2 ta = values(a), tb = values(b);
  s1 = ta.x + ta.y;
  s2 = tb.x + tb.y;
}
// g becomes dx = rstd (g - s1 - xhat s2), s1 and s2 the means over the row.
template <int VEC, int NV>
__device__ __forceinline__ void backward_out(const Row<VEC, NV>& x, Row<VEC, NV>& g, float rstd, float s1,
                                             float s2) {
  const F2 r = f2(rstd, rstd), c1 = f2(-rstd * s1, -rstd * s1), c2 = f2(-rstd * s2, -rstd * s2);
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) g.v[i] = fma2(x.v[i], c2, fma2(g.v[i], r, c1));
}
template <int VEC, int NV>
__device__ __forceinline__ void add_row(Row<VEC, NV>& a, const Row<VEC, NV>& b) {
#pragma unroll
  for (int i = 0; i < Row<VEC, NV>::kPairs; ++i) a.v[i] = add2(a.v[i], b.v[i]);
}
// The block's dw and db into part[2][dims].  Lanes of a warp that share columns
// add by shuffles, warps through columns[warps][2][dims] in shared memory.
template <int VEC, int NV, class Step>
__device__ __forceinline__ void leave_partials(Row<VEC, NV>& dw, Row<VEC, NV>& db, int first, Step step,
                                               int tpr, int nvec, int dims, float* columns, float* part) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float* const to = tpr <= 32 ? columns + warp * 2 * dims : part;
#pragma unroll
  for (int e = 0; e < VEC * NV; ++e) {
    const float2 w2 = values(dw.v[e / 2]), b2 = values(db.v[e / 2]);
    float w = e & 1 ? w2.y : w2.x, b = e & 1 ? b2.y : b2.x;
    for (int o = tpr; o < 32; o <<= 1) {
      w += __shfl_xor_sync(kFull, w, o);
      b += __shfl_xor_sync(kFull, b, o);
    }
    const int q = first + e / VEC * step;
    if (q < nvec && (tpr > 32 || int(threadIdx.x & 31) < tpr)) {
      to[q * VEC + e % VEC] = w;
      to[dims + q * VEC + e % VEC] = b;
    }
  }
  if (tpr > 32) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * dims; i += blockDim.x) {
    float s = 0.0f;
#pragma unroll 8
    for (int w = 0; w < warps; ++w) s += columns[w * 2 * dims + i];
    part[i] = s;
  }
}

// ---- plain loads ----
template <class T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : kWarpRowThreads)
layer_norm_kernel(LayerNormArgs a, int tpr_) {
  __shared__ float2 sums[32];
  RowSum rs{sums};
  const int tpr = BLOCK ? int(blockDim.x) : tpr_;
  const int lane = BLOCK ? int(threadIdx.x) : int(threadIdx.x) & (tpr - 1);
  const int per_block = BLOCK ? 1 : int(blockDim.x) / tpr;
  const int in_block = BLOCK ? 0 : int(threadIdx.x) / tpr;
  const int nvec = a.dims / VEC;
  const float inv_n = 1.0f / float(a.dims);
  Row<VEC, NV> w, b;
  load_parameter<T>(a.weight, lane, tpr, nvec, 1.0f, w);
  load_parameter<T>(a.bias, lane, tpr, nvec, 0.0f, b);
  for (int64_t base = int64_t(blockIdx.x) * per_block; base < a.rows;
       base += int64_t(gridDim.x) * per_block) {
    const int64_t row = base + in_block;
    const bool active = row < a.rows;
    Row<VEC, NV> x;
    load_row<T>(static_cast<const T*>(a.x) + row * a.x_stride, lane, tpr, nvec, active, x);
    const float mean = row_sum<BLOCK>(rs, tpr, forward_sum(x)) * inv_n;
    const float var = row_sum<BLOCK>(rs, tpr, forward_centre(x, mean, lane, tpr, nvec)) * inv_n;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (!active) continue;
    forward_out(x, rstd, w, b);
    store_row<T>(static_cast<T*>(a.y) + row * a.y_stride, lane, tpr, nvec, x);
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

template <class T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : kWarpRowThreads)
layer_norm_backward_kernel(LayerNormBackwardArgs a, int tpr_) {
  let_next_launch();
  __shared__ float2 sums[32];
  extern __shared__ float columns[];  // [warps][2][dims], rows of a warp or less
  RowSum rs{sums};
  const int tpr = BLOCK ? int(blockDim.x) : tpr_;
  const int lane = BLOCK ? int(threadIdx.x) : int(threadIdx.x) & (tpr - 1);
  const int per_block = BLOCK ? 1 : int(blockDim.x) / tpr;
  const int in_block = BLOCK ? 0 : int(threadIdx.x) / tpr;
  const int nvec = a.dims / VEC;
  const float inv_n = 1.0f / float(a.dims);
  const bool params = a.partials != nullptr;
  Row<VEC, NV> w, dw{}, db{};
  load_parameter<T>(a.weight, lane, tpr, nvec, 1.0f, w);
  for (int64_t base = int64_t(blockIdx.x) * per_block; base < a.rows;
       base += int64_t(gridDim.x) * per_block) {
    const int64_t row = base + in_block;
    const bool active = row < a.rows;
    Row<VEC, NV> x, g;
    load_row<T>(static_cast<const T*>(a.x) + row * a.x_stride, lane, tpr, nvec, active, x);
    load_row<T>(static_cast<const T*>(a.dy) + row * a.dy_stride, lane, tpr, nvec, active, g);
    const float mean = active ? a.mean[row] : 0.0f, rstd = active ? a.rstd[row] : 0.0f;
    float s1, s2;
    backward_sums<T>(x, g, w, mean, rstd, params, dw, db, s1, s2);
    row_sum2<BLOCK>(rs, tpr, s1, s2);
    if (!active || !a.dx) continue;
    backward_out(x, g, rstd, s1 * inv_n, s2 * inv_n);
    if (a.residual) {
      load_row<T>(static_cast<const T*>(a.residual) + row * a.residual_stride, lane, tpr, nvec, true, x);
      add_row(g, x);
    }
    store_row<T>(static_cast<T*>(a.dx) + row * a.dx_stride, lane, tpr, nvec, g);
  }
  if (params)
    leave_partials(dw, db, lane, tpr, tpr, nvec, a.dims, columns,
                   a.partials + int64_t(blockIdx.x) * 2 * a.dims);
}

// ---- bulk copies: rows in flight ahead of the arithmetic ----
__device__ unsigned long long g_timeouts = 0;  // bounded waits that gave up

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(dst), "r"(src),
               "r"(bytes)
               : "memory");
}

// A warp's ring: `stages` slots of `slot` bytes, one barrier each.
struct WarpRing {
  uint32_t bars, data, slot;
  int stages;
  __device__ __forceinline__ uint32_t bar(int s) const { return bars + 8 * s; }
  __device__ __forceinline__ uint32_t at(int s) const { return data + s * slot; }
};
__device__ __forceinline__ WarpRing warp_ring(char* smem, int stages, uint32_t slot) {
  // barriers of all warps first, then the slots
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t base = tc::smem_addr(smem);
  WarpRing r;
  r.bars = base + warp * stages * 8;
  r.data = base + ((warps * stages * 8 + 127) & ~127) + uint32_t(warp) * stages * slot;
  r.slot = slot;
  r.stages = stages;
  if ((threadIdx.x & 31) == 0) {
    for (int s = 0; s < stages; ++s) tc::bar_init(r.bar(s), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  return r;
}

// Plain copies of a last tile with fewer than eight rows.
template <class T>
__device__ __forceinline__ void copy_in(char* dst, const T* src, int count, int lane) {
  for (int i = lane; i < count; i += 32) reinterpret_cast<T*>(dst)[i] = src[i];
}
template <class T>
__device__ __forceinline__ void copy_out(T* dst, const char* src, int count, int lane) {
  for (int i = lane; i < count; i += 32) dst[i] = reinterpret_cast<const T*>(src)[i];
}

// What one warp of the tile kernels walks: tiles of `rows` (a multiple of four)
// rows, a whole number of 16-byte units whatever the width.
struct TileShape {
  int tpr, stages, rows;
};

template <class T, int VEC, int NV>
__global__ void __launch_bounds__(256, 2) layer_norm_tiles_kernel(LayerNormArgs a, TileShape shape) {
  extern __shared__ __align__(128) char smem[];
  const int tpr = shape.tpr, stages = shape.stages, tile_rows = shape.rows;
  const uint32_t base = tc::smem_addr(smem);
  const uint32_t tile_bytes = tile_rows * a.dims * sizeof(T);
  const WarpRing ring = warp_ring(smem, stages, (tile_bytes + 127) & ~127u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane & (tpr - 1), group = lane / tpr, at_once = 32 / tpr;
  const int nvec = a.dims / VEC;
  const float inv_n = 1.0f / float(a.dims);
  const int64_t tiles = (a.rows + tile_rows - 1) / tile_rows;
  const int64_t full_tiles = a.rows / tile_rows;
  const int64_t first = int64_t(blockIdx.x) * (blockDim.x >> 5) + warp;
  const int64_t step = int64_t(gridDim.x) * (blockDim.x >> 5);
  const T* const x = static_cast<const T*>(a.x);
  T* const y = static_cast<T*>(a.y);
  RowSum none{};

  auto request = [&](int64_t tile, int slot) {  // lane 0
    if (tile < full_tiles) {
      tc::bar_expect(ring.bar(slot), tile_bytes);
      bulk_load(ring.at(slot), x + tile * tile_rows * a.dims, tile_bytes, ring.bar(slot));
    }
  };
  if (lane == 0)
    for (int s = 0; s < stages - 1; ++s) request(first + s * step, s);
  Row<VEC, NV> w, b;
  load_parameter<T>(a.weight, sub * NV, Next(), nvec, 1.0f, w);
  load_parameter<T>(a.bias, sub * NV, Next(), nvec, 0.0f, b);
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t tile = first; tile < tiles; tile += step) {
    char* const at = smem + (ring.at(slot) - base);
    const int rows = int(min(int64_t(tile_rows), a.rows - tile * tile_rows));
    if (rows == tile_rows) {
      ok = __all_sync(kFull, tc::bar_wait(ring.bar(slot), phase));
      if (!ok) break;
      if (lane == 0) {
        // the slot before this one, once its results have left, takes a tile
        // that arrives under this one's arithmetic
        tc::bulk_wait_read<0>();
        request(tile + (stages - 1) * step, slot == 0 ? stages - 1 : slot - 1);
      }
    } else {
      if (lane == 0) tc::bulk_wait_read<0>();
      __syncwarp();
      copy_in<T>(at, x + tile * tile_rows * a.dims, rows * a.dims, lane);
      __syncwarp();
    }
    for (int r0 = 0; r0 < tile_rows; r0 += at_once) {
      const int r = r0 + group;
      T* const row = reinterpret_cast<T*>(at) + r * a.dims;
      Row<VEC, NV> v;
      load_row<T>(row, sub * NV, Next(), nvec, r < rows, v);
      const float mean = row_sum<false>(none, tpr, forward_sum(v)) * inv_n;
      const float var = row_sum<false>(none, tpr, forward_centre(v, mean, sub * NV, Next(), nvec)) * inv_n;
      const float rstd = 1.0f / sqrtf(var + a.eps);
      if (r < rows) {
        forward_out(v, rstd, w, b);
        store_row<T>(row, sub * NV, Next(), nvec, v);
        if (sub == 0) {
          if (a.mean) a.mean[tile * tile_rows + r] = mean;
          if (a.rstd) a.rstd[tile * tile_rows + r] = rstd;
        }
      }
    }
    if (rows == tile_rows) {
      tc::fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        bulk_store(y + tile * tile_rows * a.dims, ring.at(slot), tile_bytes);
        tc::bulk_commit();
      }
    } else {
      __syncwarp();
      copy_out<T>(y + tile * tile_rows * a.dims, at, rows * a.dims, lane);
    }
    if (++slot == stages) {
      slot = 0;
      phase ^= 1;
    }
  }
  if (lane == 0) tc::bulk_wait_all();
  if (!ok && lane == 0) {
    atomicAdd(&g_timeouts, 1ull);
    // copies in flight must land before the block may leave
    for (int s = 0; s < stages; ++s) tc::bar_wait(ring.bar(s), s < slot ? phase ^ 1 : phase);
  }
}

// The slots of the backward ring: x (dx in place), dy, residual, mean, rstd.
__host__ __device__ inline uint32_t backward_slot(uint32_t tile_bytes, bool residual, int tile_rows) {
  return ((residual ? 3 : 2) * tile_bytes + 2 * tile_rows * 4 + 127) & ~127u;
}

// Blocks of eight warps that an SM's registers are to hold.
constexpr int kBackwardBlocks = 2;

template <class T, int VEC, int NV>
__global__ void __launch_bounds__(256, kBackwardBlocks)
layer_norm_backward_tiles_kernel(LayerNormBackwardArgs a, TileShape shape) {
  let_next_launch();
  extern __shared__ __align__(128) char smem[];
  const int tpr = shape.tpr, stages = shape.stages, tile_rows = shape.rows;
  const uint32_t base = tc::smem_addr(smem);
  const uint32_t tile_bytes = tile_rows * a.dims * sizeof(T);
  const WarpRing ring =
      warp_ring(smem, stages, backward_slot(tile_bytes, a.residual != nullptr, tile_rows));
  const uint32_t stats = (a.residual ? 3 : 2) * tile_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int sub = lane & (tpr - 1), group = lane / tpr, at_once = 32 / tpr;
  const int nvec = a.dims / VEC;
  const float inv_n = 1.0f / float(a.dims);
  const int64_t tiles = (a.rows + tile_rows - 1) / tile_rows;
  const int64_t full_tiles = a.rows / tile_rows;
  const int64_t first = int64_t(blockIdx.x) * warps + warp;
  const int64_t step = int64_t(gridDim.x) * warps;
  const T* const x = static_cast<const T*>(a.x);
  const T* const dy = static_cast<const T*>(a.dy);
  const T* const res = static_cast<const T*>(a.residual);
  T* const dx = static_cast<T*>(a.dx);
  const bool params = a.partials != nullptr;
  RowSum none{};

  auto request = [&](int64_t tile, int slot) {  // lane 0
    if (tile < full_tiles) {
      const int64_t row = tile * tile_rows, from = row * a.dims;
      const uint32_t bar = ring.bar(slot), at = ring.at(slot);
      tc::bar_expect(bar, stats + 2 * tile_rows * 4);
      bulk_load(at, x + from, tile_bytes, bar);
      bulk_load(at + tile_bytes, dy + from, tile_bytes, bar);
      if (res) bulk_load(at + 2 * tile_bytes, res + from, tile_bytes, bar);
      bulk_load(at + stats, a.mean + row, tile_rows * 4, bar);
      bulk_load(at + stats + tile_rows * 4, a.rstd + row, tile_rows * 4, bar);
    }
  };
  if (lane == 0)
    for (int s = 0; s < stages - 1; ++s) request(first + s * step, s);
  Row<VEC, NV> w, dw{}, db{};
  load_parameter<T>(a.weight, sub * NV, Next(), nvec, 1.0f, w);
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t tile = first; tile < tiles; tile += step) {
    char* const at = smem + (ring.at(slot) - base);
    const int64_t from = tile * tile_rows * a.dims;
    const int rows = int(min(int64_t(tile_rows), a.rows - tile * tile_rows));
    if (rows == tile_rows) {
      ok = __all_sync(kFull, tc::bar_wait(ring.bar(slot), phase));
      if (!ok) break;
      if (lane == 0) {
        // as in the forward kernel
        tc::bulk_wait_read<0>();
        request(tile + (stages - 1) * step, slot == 0 ? stages - 1 : slot - 1);
      }
    } else {
      if (lane == 0) tc::bulk_wait_read<0>();
      __syncwarp();
      copy_in<T>(at, x + from, rows * a.dims, lane);
      copy_in<T>(at + tile_bytes, dy + from, rows * a.dims, lane);
      if (res) copy_in<T>(at + 2 * tile_bytes, res + from, rows * a.dims, lane);
      copy_in<float>(at + stats, a.mean + tile * tile_rows, rows, lane);
      copy_in<float>(at + stats + tile_rows * 4, a.rstd + tile * tile_rows, rows, lane);
      __syncwarp();
    }
    const float* const st = reinterpret_cast<const float*>(at + stats);
    for (int r0 = 0; r0 < tile_rows; r0 += at_once) {
      const int r = r0 + group;
      const bool active = r < rows;
      T* const row = reinterpret_cast<T*>(at) + r * a.dims;
      const T* const grow = row + tile_rows * a.dims;
      const float mean = active ? st[r] : 0.0f, rstd = active ? st[tile_rows + r] : 0.0f;
      Row<VEC, NV> xh, g;
      load_row<T>(row, sub * NV, Next(), nvec, active, xh);
      load_row<T>(grow, sub * NV, Next(), nvec, active, g);
      float s1, s2;
      backward_sums<T>(xh, g, w, mean, rstd, params, dw, db, s1, s2);
      row_sum2<false>(none, tpr, s1, s2);
      if (!dx || !active) continue;
      backward_out(xh, g, rstd, s1 * inv_n, s2 * inv_n);
      if (res) {
        load_row<T>(grow + tile_rows * a.dims, sub * NV, Next(), nvec, true, xh);
        add_row(g, xh);
      }
      store_row<T>(row, sub * NV, Next(), nvec, g);
    }
    if (rows == tile_rows) {
      tc::fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        if (dx) bulk_store(dx + from, ring.at(slot), tile_bytes);
        tc::bulk_commit();
      }
    } else {
      __syncwarp();
      if (dx) copy_out<T>(dx + from, at, rows * a.dims, lane);
    }
    if (++slot == stages) {
      slot = 0;
      phase ^= 1;
    }
  }
  if (lane == 0) tc::bulk_wait_all();
  if (!ok && lane == 0) {
    atomicAdd(&g_timeouts, 1ull);
    for (int s = 0; s < stages; ++s) tc::bar_wait(ring.bar(s), s < slot ? phase ^ 1 : phase);
  }
  if (!params) return;
  __syncthreads();  // the ring's memory now holds the block's columns
  leave_partials(dw, db, sub * NV, Next(), tpr, nvec, a.dims,
                 reinterpret_cast<float*>(smem + ((warps * stages * 8 + 127) & ~127)),
                 a.partials + int64_t(blockIdx.x) * 2 * a.dims);
}

// ---- wide rows: a block per row, rows copied ahead ----
template <class T, int NV>
__global__ void __launch_bounds__(512) layer_norm_wide_kernel(LayerNormArgs a, int stages) {
  constexpr int VEC = 16 / int(sizeof(T));
  extern __shared__ __align__(128) char smem[];
  __shared__ float2 sums[32];
  __shared__ uint64_t bars[8];
  __shared__ int gave_up[2];  // by the parity of the row's turn
  RowSum rs{sums};
  const int nvec = a.dims / VEC, threads = blockDim.x, lane = threadIdx.x;
  const uint32_t row_bytes = a.dims * sizeof(T), slot_bytes = (row_bytes + 127) & ~127u;
  const uint32_t base = tc::smem_addr(smem), bar0 = tc::smem_addr(bars);
  const float inv_n = 1.0f / float(a.dims);
  const T* const x = static_cast<const T*>(a.x);
  if (lane == 0) {
    gave_up[0] = gave_up[1] = 0;
    for (int s = 0; s < stages; ++s) tc::bar_init(bar0 + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  auto request = [&](int64_t row, int slot) {  // thread 0
    if (row < a.rows) {
      tc::bar_expect(bar0 + 8 * slot, row_bytes);
      bulk_load(base + slot * slot_bytes, x + row * a.x_stride, row_bytes, bar0 + 8 * slot);
    }
  };
  if (lane == 0)
    for (int s = 0; s < stages; ++s) request(blockIdx.x + int64_t(s) * gridDim.x, s);
  Row<VEC, NV> w, b;
  load_parameter<T>(a.weight, lane, threads, nvec, 1.0f, w);
  load_parameter<T>(a.bias, lane, threads, nvec, 0.0f, b);
  int slot = 0, turn = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    if (!tc::bar_wait(bar0 + 8 * slot, phase)) gave_up[turn] = 1;
    Row<VEC, NV> v;
    load_row<T>(reinterpret_cast<const T*>(smem + slot * slot_bytes), lane, threads, nvec, true, v);
    const float mean = row_sum<true>(rs, 0, forward_sum(v)) * inv_n;
    // past the barrier in row_sum every thread has read the slot
    ok = gave_up[turn] == 0;
    if (!ok) break;
    if (lane == 0) request(row + int64_t(stages) * gridDim.x, slot);
    const float var = row_sum<true>(rs, 0, forward_centre(v, mean, lane, threads, nvec)) * inv_n;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (++slot == stages) {
      slot = 0;
      phase ^= 1;
    }
    forward_out(v, rstd, w, b);
    store_row<T>(static_cast<T*>(a.y) + row * a.y_stride, lane, threads, nvec, v);
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
  if (!ok && lane == 0) {
    atomicAdd(&g_timeouts, 1ull);
    for (int s = 0; s < stages; ++s) tc::bar_wait(bar0 + 8 * s, s < slot ? phase ^ 1 : phase);
  }
}

template <class T, int NV>
__global__ void __launch_bounds__(512) layer_norm_backward_wide_kernel(LayerNormBackwardArgs a,
                                                                       int stages) {
  let_next_launch();
  constexpr int VEC = 16 / int(sizeof(T));
  extern __shared__ __align__(128) char smem[];
  __shared__ float2 sums[32];
  __shared__ uint64_t bars[8];
  __shared__ int gave_up[2];  // by the parity of the row's turn
  RowSum rs{sums};
  const int nvec = a.dims / VEC, threads = blockDim.x, lane = threadIdx.x;
  const uint32_t row_bytes = a.dims * sizeof(T), pitch = (row_bytes + 127) & ~127u;
  const uint32_t slot_bytes = (a.residual ? 3 : 2) * pitch;
  const uint32_t base = tc::smem_addr(smem), bar0 = tc::smem_addr(bars);
  const float inv_n = 1.0f / float(a.dims);
  const bool params = a.partials != nullptr;
  if (lane == 0) {
    gave_up[0] = gave_up[1] = 0;
    for (int s = 0; s < stages; ++s) tc::bar_init(bar0 + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  auto request = [&](int64_t row, int slot) {  // thread 0
    if (row < a.rows) {
      const uint32_t bar = bar0 + 8 * slot, at = base + slot * slot_bytes;
      tc::bar_expect(bar, (a.residual ? 3 : 2) * row_bytes);
      bulk_load(at, static_cast<const T*>(a.x) + row * a.x_stride, row_bytes, bar);
      bulk_load(at + pitch, static_cast<const T*>(a.dy) + row * a.dy_stride, row_bytes, bar);
      if (a.residual)
        bulk_load(at + 2 * pitch, static_cast<const T*>(a.residual) + row * a.residual_stride, row_bytes,
                  bar);
    }
  };
  if (lane == 0)
    for (int s = 0; s < stages; ++s) request(blockIdx.x + int64_t(s) * gridDim.x, s);
  Row<VEC, NV> w, dw{}, db{};
  load_parameter<T>(a.weight, lane, threads, nvec, 1.0f, w);
  int slot = 0, turn = 0;
  uint32_t phase = 0;
  bool ok = true;
  // the next row's statistics: their latency passes under this row
  float next_mean = int64_t(blockIdx.x) < a.rows ? a.mean[blockIdx.x] : 0.0f;
  float next_rstd = int64_t(blockIdx.x) < a.rows ? a.rstd[blockIdx.x] : 0.0f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    if (row + gridDim.x < a.rows) {
      next_mean = a.mean[row + gridDim.x];
      next_rstd = a.rstd[row + gridDim.x];
    }
    if (!tc::bar_wait(bar0 + 8 * slot, phase)) gave_up[turn] = 1;
    const char* const at = smem + slot * slot_bytes;
    Row<VEC, NV> xh, g;
    load_row<T>(reinterpret_cast<const T*>(at), lane, threads, nvec, true, xh);
    load_row<T>(reinterpret_cast<const T*>(at + pitch), lane, threads, nvec, true, g);
    float s1, s2;
    backward_sums<T>(xh, g, w, mean, rstd, params, dw, db, s1, s2);
    row_sum2<true>(rs, 0, s1, s2);
    ok = gave_up[turn] == 0;
    if (!ok) break;
    if (a.dx) {
      backward_out(xh, g, rstd, s1 * inv_n, s2 * inv_n);
      if (a.residual) {
        load_row<T>(reinterpret_cast<const T*>(at + 2 * pitch), lane, threads, nvec, true, xh);
        add_row(g, xh);
      }
      store_row<T>(static_cast<T*>(a.dx) + row * a.dx_stride, lane, threads, nvec, g);
    }
    // every thread has read x and dy past the barrier in row_sum2, but the
    // residual only now
    if (a.residual) __syncthreads();
    if (lane == 0) request(row + int64_t(stages) * gridDim.x, slot);
    if (++slot == stages) {
      slot = 0;
      phase ^= 1;
    }
  }
  if (!ok && lane == 0) {
    atomicAdd(&g_timeouts, 1ull);
    for (int s = 0; s < stages; ++s) tc::bar_wait(bar0 + 8 * s, s < slot ? phase ^ 1 : phase);
  }
  if (params)
    leave_partials(dw, db, lane, threads, threads, nvec, a.dims, nullptr,
                   a.partials + int64_t(blockIdx.x) * 2 * a.dims);
}

// Rows too long for registers: a block walks the row three times (the second
// and third walks find it in L2).
template <class T>
__global__ void __launch_bounds__(512) layer_norm_long_kernel(LayerNormArgs a) {
  __shared__ float2 sums[32];
  RowSum rs{sums};
  const float inv_n = 1.0f / float(a.dims);
  const T* const w = static_cast<const T*>(a.weight);
  const T* const b = static_cast<const T*>(a.bias);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* const y = static_cast<T*>(a.y) + row * a.y_stride;
    float s = 0.0f;
    for (int i = threadIdx.x; i < a.dims; i += blockDim.x) s += to_f32(x[i]);
    const float mean = row_sum<true>(rs, 0, s) * inv_n;
    float v = 0.0f;
    for (int i = threadIdx.x; i < a.dims; i += blockDim.x) {
      const float d = to_f32(x[i]) - mean;
      v += d * d;
    }
    const float rstd = 1.0f / sqrtf(row_sum<true>(rs, 0, v) * inv_n + a.eps);
    for (int i = threadIdx.x; i < a.dims; i += blockDim.x) {
      float o = (to_f32(x[i]) - mean) * rstd;
      if (w) o *= to_f32(w[i]);
      if (b) o += to_f32(b[i]);
      y[i] = from_f32<T>(o);
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

// Long rows: dx by a block per row in two walks; dw and db by
// column_partials_kernel.
template <class T>
__global__ void __launch_bounds__(512) layer_norm_backward_long_kernel(LayerNormBackwardArgs a) {
  __shared__ float2 sums[32];
  RowSum rs{sums};
  const float inv_n = 1.0f / float(a.dims);
  const T* const w = static_cast<const T*>(a.weight);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* const dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int i = threadIdx.x; i < a.dims; i += blockDim.x) {
      const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.0f);
      s1 += g;
      s2 += g * ((to_f32(x[i]) - mean) * rstd);
    }
    row_sum2<true>(rs, 0, s1, s2);
    s1 *= inv_n;
    s2 *= inv_n;
    T* const out = static_cast<T*>(a.dx) + row * a.dx_stride;
    const T* const res =
        a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    for (int i = threadIdx.x; i < a.dims; i += blockDim.x) {
      const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.0f);
      float d = rstd * (g - s1 - (to_f32(x[i]) - mean) * rstd * s2);
      if (res) d += to_f32(res[i]);
      out[i] = from_f32<T>(d);
    }
  }
}
template <class T>
__global__ void __launch_bounds__(256) column_partials_kernel(LayerNormBackwardArgs a,
                                                              int64_t rows_per_block) {
  let_next_launch();
  const int col = blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= a.dims) return;
  const int64_t begin = blockIdx.y * rows_per_block;
  const int64_t end = begin + rows_per_block < a.rows ? begin + rows_per_block : a.rows;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = begin; row < end; ++row) {
    const float g = to_f32(static_cast<const T*>(a.dy)[row * a.dy_stride + col]);
    db += g;
    if (a.dweight)
      dw += g * ((to_f32(static_cast<const T*>(a.x)[row * a.x_stride + col]) - a.mean[row]) *
                 a.rstd[row]);
  }
  float* const part = a.partials + int64_t(blockIdx.y) * 2 * a.dims;
  part[col] = dw;
  part[a.dims + col] = db;
}

// dw and db from the blocks' partial sums: 32 columns per block, whose 32 row
// lanes each add every 32nd partial in order; their sums meet in order too.
template <class T>
__global__ void __launch_bounds__(1024) column_reduce_kernel(const float* __restrict__ partials,
                                                             int count, int dims, T* dweight,
                                                             T* dbias) {
  wait_for_previous();
  __shared__ float acc[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t col = int64_t(blockIdx.x) * 32 + tx;  // over [2][dims]
  float s = 0.0f;
  if (col < 2 * int64_t(dims))
#pragma unroll 8
    for (int p = ty; p < count; p += 32) s += partials[int64_t(p) * 2 * dims + col];
  acc[ty][tx] = s;
  __syncthreads();
  // warp ty adds column ty's 32 sums
  s = acc[tx][ty];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  const int64_t out_col = int64_t(blockIdx.x) * 32 + ty;
  if (tx != 0 || out_col >= 2 * int64_t(dims)) return;
  T* const out = out_col < dims ? dweight : dbias;
  if (out) out[out_col < dims ? out_col : out_col - dims] = from_f32<T>(s);
}

// How a row is spread over threads, in accesses of `vec` values.
struct RowPlan {
  int vec;
  int nv;      // accesses per thread; 0: the long kernel
  int tpr;     // threads per row
  bool block;  // the whole block has one row
};

bool aligned(const void* p, int64_t stride, size_t sz, int vec) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (sz * vec) == 0 && stride % vec == 0);
}

// Accesses per thread at most (16 to 20 values, which the backward kernels hold
// four times over: xhat, g, dw, db), and the number aimed at where a warp's
// lanes have a row.
int aimed_accesses(int vec) { return vec == 8 ? 2 : vec == 4 ? 3 : vec == 2 ? 5 : 9; }
int most_accesses(int vec) { return vec == 8 ? 2 : vec == 4 ? 5 : vec == 2 ? 9 : 16; }

// Lanes of a warp to a row, or nv = 0 where a warp cannot hold it.  Few lanes
// with many values each: fewer shuffle steps and address computations per
// value (130 columns: 8 lanes with nine pairs).
RowPlan plan_lanes(int dims, int vec) {
  RowPlan p{};
  p.vec = vec;
  const int nvec = dims / vec, most = most_accesses(vec);
  p.tpr = nvec >= 8 ? 8 : 4;
  while (p.tpr < 32 && (nvec + p.tpr - 1) / p.tpr > aimed_accesses(vec)) p.tpr *= 2;
  const int nv = (nvec + p.tpr - 1) / p.tpr;
  p.nv = nv <= most ? nv : 0;
  return p;
}
// A warp's lanes or a block for rows that are read with plain loads.
RowPlan plan_row(int dims, int vec) {
  RowPlan p = plan_lanes(dims, vec);
  if (p.nv) return p;
  p.block = true;
  const int nvec = dims / vec, most = most_accesses(vec);
  for (int nv = 1; nv <= most; ++nv) {
    const int threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
    if (threads > 512) continue;
    p.nv = nv;
    p.tpr = threads;
    if (threads <= 256) break;
  }
  return p;
}

// Calls f(integral_constant<VEC>, integral_constant<NV>) with the smallest
// instance that has room for nv accesses.
template <class T, class F>
auto with_row_shape(int vec, int nv, F&& f) {
  using std::integral_constant;
  if (vec == 1) {
    if (nv <= 2) return f(integral_constant<int, 1>(), integral_constant<int, 2>());
    if (nv <= 5) return f(integral_constant<int, 1>(), integral_constant<int, 5>());
    if (nv <= 9) return f(integral_constant<int, 1>(), integral_constant<int, 9>());
    return f(integral_constant<int, 1>(), integral_constant<int, 16>());
  }
  if (vec == 2) {
    if (nv <= 2) return f(integral_constant<int, 2>(), integral_constant<int, 2>());
    if (nv <= 5) return f(integral_constant<int, 2>(), integral_constant<int, 5>());
    return f(integral_constant<int, 2>(), integral_constant<int, 9>());
  }
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) {
      if (nv <= 1) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
      return f(integral_constant<int, 8>(), integral_constant<int, 2>());
    }
  }
  if (nv <= 2) return f(integral_constant<int, 4>(), integral_constant<int, 2>());
  if (nv <= 3) return f(integral_constant<int, 4>(), integral_constant<int, 3>());
  return f(integral_constant<int, 4>(), integral_constant<int, 5>());
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  return sms;
}

constexpr int kLongSplits = 64;        // row ranges of column_partials_kernel
constexpr int kMaxPartials = 148 * 8;  // blocks that leave partial sums

template <class T, int VEC, int NV>
void forward_launch(const LayerNormArgs& a, const RowPlan& p, cudaStream_t stream) {
  if (p.block) {
    const int64_t grid = std::min<int64_t>(a.rows, int64_t(sm_count()) * (2048 / p.tpr));
    layer_norm_kernel<T, VEC, NV, true><<<unsigned(grid), p.tpr, 0, stream>>>(a, p.tpr);
  } else {
    const int per_block = kWarpRowThreads / p.tpr;
    const int64_t grid =
        std::min<int64_t>((a.rows + per_block - 1) / per_block, int64_t(sm_count()) * 8 * 4);
    layer_norm_kernel<T, VEC, NV, false><<<unsigned(grid), kWarpRowThreads, 0, stream>>>(a, p.tpr);
  }
}

template <class T, int VEC, int NV>
int backward_launch(const LayerNormBackwardArgs& a, const RowPlan& p, cudaStream_t stream) {
  if (p.block) {
    const int64_t grid = std::min<int64_t>(std::min<int64_t>(a.rows, kMaxPartials),
                                           int64_t(sm_count()) * (1024 / p.tpr));
    layer_norm_backward_kernel<T, VEC, NV, true>
        <<<unsigned(grid), p.tpr, 0, stream>>>(a, p.tpr);
    return int(grid);
  }
  const int per_block = kWarpRowThreads / p.tpr;
  const int64_t grid =
      std::min<int64_t>(std::min<int64_t>((a.rows + per_block - 1) / per_block, kMaxPartials),
                        int64_t(sm_count()) * 4);
  const size_t smem =
      a.partials ? size_t(kWarpRowThreads / 32) * a.dims * 2 * sizeof(float) : 0;
  layer_norm_backward_kernel<T, VEC, NV, false>
      <<<unsigned(grid), kWarpRowThreads, smem, stream>>>(a, p.tpr);
  return int(grid);
}

bool bulk_rows(const void* p, int64_t stride, size_t size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * int64_t(size) % 16 == 0);
}
bool gapless(const void* p, int64_t stride, int64_t rows, int dims) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride == dims || rows <= 1));
}

constexpr size_t kSmemPerSm = 220 * 1024;

// The tile ring's shape, or row.nv = 0 where a tile has no place.
struct TilePlan {
  RowPlan row;
  int warps, stages, tile_rows;
  size_t smem;
  TileShape shape() const { return {row.tpr, stages, tile_rows}; }
};
// slot_of(tile_rows): bytes of one ring slot.
template <class F>
TilePlan plan_tiles(size_t size, int dims, int64_t rows, int most_blocks, bool deep, F&& slot_of) {
  TilePlan p{};
  int vec = 16 / int(size);
  while (dims % vec) vec /= 2;
  const RowPlan row = plan_lanes(dims, vec);
  if (row.nv == 0) return p;
  // most_blocks blocks of eight warps fit an SM's registers.  Tiles of eight
  // rows (or more) where their rings leave room for all, else of four where those are
  // whole 16-byte units and a warp has no more rows at once.
  // Narrow rows take more to a tile: 2 KB keep the copies' count down
  // (885704 x 8 bf16 backward: 61 us with tiles of 128 bytes).
  int whole = 8;
  while (whole < 64 && size_t(dims) * size * whole < 2048 && rows / (2 * whole) >= 148 * 16) whole *= 2;
  const int most_stages = deep ? 5 : 4;
  const bool four_first = deep && size_t(dims) * size * 4 >= 2048;
  for (int tile_rows : {four_first ? 4 : whole, four_first ? whole : 4}) {
    if (tile_rows == 4 && (size_t(dims) * size * 4 % 16 || row.tpr < 8)) continue;
    const size_t slot = slot_of(tile_rows);
    // few tiles: fewer warps to a block, so that every SM has some
    const int64_t tiles = (rows + tile_rows - 1) / tile_rows;
    int warps = 8;
    while (warps > 1 && tiles < int64_t(warps) * 148) warps /= 2;
    for (int blocks = most_blocks * (8 / warps); blocks >= 1; --blocks) {
      const int stages =
          int(std::min<size_t>(most_stages, kSmemPerSm / blocks / (size_t(warps) * (slot + 8) + 128)));
      if (stages < 2) continue;
      if (p.row.nv && blocks < most_blocks) break;  // eight rows fit as well as four
      p.smem = ((size_t(warps) * stages * 8 + 127) & ~size_t(127)) + size_t(warps) * stages * slot;
      p.smem = (p.smem + 4095) & ~size_t(4095);  // few distinct launch shapes
      p.row = row;
      p.warps = warps;
      p.stages = stages;
      p.tile_rows = tile_rows;
      if (blocks >= most_blocks) return p;
      break;
    }
  }
  return p;
}
template <class K>
npa_status tile_grid(K kernel, const TilePlan& p, int64_t rows, unsigned* grid) {
  int per_sm = 0, sms = 0;
  NPA_TRY(kernel_occupancy(reinterpret_cast<const void*>(kernel), p.warps * 32, p.smem, &per_sm, &sms));
  if (per_sm < 1) return fail(NPA_ERR_UNSUPPORTED, "layer norm kernel cannot be resident");
  const int64_t tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  *grid = unsigned(std::min<int64_t>(
      std::min<int64_t>((tiles + p.warps - 1) / p.warps, int64_t(per_sm) * sms), kMaxPartials));
  return NPA_OK;
}

// Wide rows: 16-byte accesses, NV of them per thread.
struct WidePlan {
  int nv, threads, stages;
  size_t smem;
};
WidePlan plan_wide(size_t size, int dims, size_t slot, int most) {
  WidePlan p{};
  const int vec = 16 / int(size), nvec = dims / vec;
  if (dims % vec || nvec < 64) return p;
  for (int nv = most; nv >= 1; nv /= 2) {
    p.threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
    p.nv = nv;
    if (p.threads >= 128) break;
  }
  if (p.threads > 512) return WidePlan{};
  const int blocks = std::max(1, 768 / p.threads);
  p.stages = int(std::min<size_t>(6, std::max<size_t>(2, kSmemPerSm / (blocks * slot))));
  p.smem = (p.stages * slot + 4095) & ~size_t(4095);  // few distinct launch shapes
  return p.smem <= kSmemPerSm ? p : WidePlan{};
}
template <class K>
npa_status wide_grid(K kernel, const WidePlan& p, int64_t rows, unsigned* grid) {
  int per_sm = 0, sms = 0;
  NPA_TRY(kernel_occupancy(reinterpret_cast<const void*>(kernel), p.threads, p.smem, &per_sm, &sms));
  if (per_sm < 1) return fail(NPA_ERR_UNSUPPORTED, "layer norm kernel cannot be resident");
  *grid = unsigned(std::min<int64_t>(std::min<int64_t>(rows, kMaxPartials), int64_t(per_sm) * sms));
  return NPA_OK;
}

template <class T>
npa_status forward_typed(const LayerNormArgs& a, cudaStream_t s) {
  if (gapless(a.x, a.x_stride, a.rows, a.dims) && gapless(a.y, a.y_stride, a.rows, a.dims)) {
    // f32 rows of 256 to 576 bytes keep five tiles to a ring, of four rows from 512
    // bytes on (536 MB of x in six places each, median us without and with it: 64
    // values 209, 171; 66 179, 177; 68 194, 198; 72 to 120 the same within 0.5 %; 128
    // 199, 181; 130 204, 175; 136 205, 168; 144 205, 195).  Elsewhere this loses: 32
    // f32 values 208, 256; 152 201, 202; 176 194, 201; 192 188, 197; 64 16-bit values
    // 213, 262; 129, an odd width, 169, 192.
    const size_t row_bytes = size_t(a.dims) * sizeof(T);
    const bool deep = sizeof(T) == 4 && a.dims % 2 == 0 && row_bytes >= 256 && row_bytes <= 576;
    const TilePlan p = plan_tiles(sizeof(T), a.dims, a.rows, 2, deep, [&](int tile_rows) {
      return (size_t(a.dims) * tile_rows * sizeof(T) + 127) & ~size_t(127);
    });
    if (p.row.nv)
      return with_row_shape<T>(p.row.vec, p.row.nv, [&](auto vec, auto nv) -> npa_status {
        const auto kernel = layer_norm_tiles_kernel<T, vec(), nv()>;
        unsigned grid = 0;
        NPA_TRY(tile_grid(kernel, p, a.rows, &grid));
        kernel<<<grid, p.warps * 32, p.smem, s>>>(a, p.shape());
        return after_launch("layer_norm_tiles_kernel");
      });
  }
  if (bulk_rows(a.x, a.x_stride, sizeof(T)) && bulk_rows(a.y, a.y_stride, sizeof(T)) &&
      bulk_rows(a.weight, 0, sizeof(T)) && bulk_rows(a.bias, 0, sizeof(T))) {
    const size_t slot = (size_t(a.dims) * sizeof(T) + 127) & ~size_t(127);
    const WidePlan p = plan_wide(sizeof(T), a.dims, slot, sizeof(T) == 2 ? 2 : 4);
    if (p.nv) {
      auto launch = [&](auto kernel) -> npa_status {
        unsigned grid = 0;
        NPA_TRY(wide_grid(kernel, p, a.rows, &grid));
        kernel<<<grid, p.threads, p.smem, s>>>(a, p.stages);
        return after_launch("layer_norm_wide_kernel");
      };
      if (p.nv == 1) return launch(layer_norm_wide_kernel<T, 1>);
      if (p.nv == 2) return launch(layer_norm_wide_kernel<T, 2>);
      if constexpr (sizeof(T) == 4) return launch(layer_norm_wide_kernel<T, 4>);
    }
  }
  int vec = 16 / int(sizeof(T));
  while (vec > 1 && (a.dims % vec || !aligned(a.x, a.x_stride, sizeof(T), vec) ||
                     !aligned(a.y, a.y_stride, sizeof(T), vec) ||
                     !aligned(a.weight, 0, sizeof(T), vec) || !aligned(a.bias, 0, sizeof(T), vec)))
    vec /= 2;
  const RowPlan p = plan_row(a.dims, vec);
  if (p.nv == 0) {
    const int64_t grid = std::min<int64_t>(a.rows, int64_t(sm_count()) * 4);
    layer_norm_long_kernel<T><<<unsigned(grid), 512, 0, s>>>(a);
    return after_launch("layer_norm_long_kernel");
  }
  with_row_shape<T>(p.vec, p.nv, [&](auto v, auto nv) {
    forward_launch<T, v(), nv()>(a, p, s);
    return 0;
  });
  return after_launch("layer_norm_kernel");
}

// The gradient kernels over the rows; *parts: partial sums left for dw and db.
template <class T>
npa_status backward_rows(const LayerNormBackwardArgs& a, int* parts, cudaStream_t s) {
  const bool params = a.partials != nullptr;
  if (gapless(a.x, a.x_stride, a.rows, a.dims) && gapless(a.dy, a.dy_stride, a.rows, a.dims) &&
      gapless(a.dx, a.dx_stride, a.rows, a.dims) &&
      gapless(a.residual, a.residual_stride, a.rows, a.dims) && bulk_rows(a.mean, 0, 4) &&
      bulk_rows(a.rstd, 0, 4)) {
    const TilePlan p = plan_tiles(sizeof(T), a.dims, a.rows, kBackwardBlocks, false, [&](int tile_rows) {
      return backward_slot(uint32_t(a.dims * tile_rows * sizeof(T)), a.residual != nullptr, tile_rows);
    });
    if (p.row.nv)
      return with_row_shape<T>(p.row.vec, p.row.nv, [&](auto vec, auto nv) -> npa_status {
        const auto kernel = layer_norm_backward_tiles_kernel<T, vec(), nv()>;
        unsigned grid = 0;
        NPA_TRY(tile_grid(kernel, p, a.rows, &grid));
        kernel<<<grid, p.warps * 32, p.smem, s>>>(a, p.shape());
        *parts = int(grid);
        return after_launch("layer_norm_backward_tiles_kernel");
      });
  }
  if (bulk_rows(a.x, a.x_stride, sizeof(T)) && bulk_rows(a.dy, a.dy_stride, sizeof(T)) &&
      bulk_rows(a.dx, a.dx_stride, sizeof(T)) && bulk_rows(a.weight, 0, sizeof(T)) &&
      bulk_rows(a.residual, a.residual_stride, sizeof(T))) {
    const size_t slot =
        (a.residual ? 3 : 2) * ((size_t(a.dims) * sizeof(T) + 127) & ~size_t(127));
    const WidePlan p = plan_wide(sizeof(T), a.dims, slot, sizeof(T) == 2 ? 2 : 4);
    if (p.nv) {
      auto launch = [&](auto kernel) -> npa_status {
        unsigned grid = 0;
        NPA_TRY(wide_grid(kernel, p, a.rows, &grid));
        kernel<<<grid, p.threads, p.smem, s>>>(a, p.stages);
        *parts = int(grid);
        return after_launch("layer_norm_backward_wide_kernel");
      };
      if (p.nv == 1) return launch(layer_norm_backward_wide_kernel<T, 1>);
      if (p.nv == 2) return launch(layer_norm_backward_wide_kernel<T, 2>);
      if constexpr (sizeof(T) == 4) return launch(layer_norm_backward_wide_kernel<T, 4>);
    }
  }
  int vec = 16 / int(sizeof(T));
  while (vec > 1 &&
         (a.dims % vec || !aligned(a.x, a.x_stride, sizeof(T), vec) ||
          !aligned(a.dy, a.dy_stride, sizeof(T), vec) ||
          !aligned(a.dx, a.dx_stride, sizeof(T), vec) || !aligned(a.weight, 0, sizeof(T), vec) ||
          !aligned(a.residual, a.residual_stride, sizeof(T), vec)))
    vec /= 2;
  const RowPlan p = plan_row(a.dims, vec);
  if (p.nv == 0) {
    if (a.dx) {
      const int64_t grid = std::min<int64_t>(a.rows, int64_t(sm_count()) * 4);
      layer_norm_backward_long_kernel<T><<<unsigned(grid), 512, 0, s>>>(a);
      NPA_TRY(after_launch("layer_norm_backward_long_kernel"));
    }
    if (params) {
      *parts = int(std::min<int64_t>(a.rows, kLongSplits));
      const int64_t per = (a.rows + *parts - 1) / *parts;
      *parts = int((a.rows + per - 1) / per);
      column_partials_kernel<T>
          <<<dim3(unsigned((a.dims + 255) / 256), unsigned(*parts)), 256, 0, s>>>(a, per);
      NPA_TRY(after_launch("column_partials_kernel"));
    }
    return NPA_OK;
  }
  *parts = with_row_shape<T>(p.vec, p.nv, [&](auto v, auto nv) -> int {
    return backward_launch<T, v(), nv()>(a, p, s);
  });
  return after_launch("layer_norm_backward_kernel");
}

template <class T>
npa_status backward_typed(LayerNormBackwardArgs a, cudaStream_t s) {
  const bool params = a.dweight || a.dbias;
  if (!params) a.partials = nullptr;
  int parts = 0;
  if (a.rows > 0 && (a.dx || params)) NPA_TRY(backward_rows<T>(a, &parts, s));
  if (!params) return NPA_OK;
  // behind a kernel of this call unless there were no rows
  NPA_CUDA(launch_kernel(parts > 0, column_reduce_kernel<T>,
                         dim3(unsigned((2 * int64_t(a.dims) + 31) / 32)), 1024, 0, s, a.partials, parts,
                         a.dims, static_cast<T*>(a.dweight), static_cast<T*>(a.dbias)),
           "column_reduce_kernel");
  return after_launch("column_reduce_kernel");
}

}  // namespace

size_t layer_norm_backward_workspace(int64_t rows, int dims) {
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(rows, kMaxPartials));
  return size_t(parts) * 2 * size_t(dims) * sizeof(float);
}

npa_status launch_layer_norm(int dtype, const LayerNormArgs& a, cudaStream_t stream) {
  switch (dtype) {
    case NPA_DTYPE_F32: return forward_typed<float>(a, stream);
    case NPA_DTYPE_F16: return forward_typed<__half>(a, stream);
    default: return forward_typed<__nv_bfloat16>(a, stream);
  }
}

npa_status launch_layer_norm_backward(int dtype, const LayerNormBackwardArgs& a,
                                      cudaStream_t stream) {
  switch (dtype) {
    case NPA_DTYPE_F32: return backward_typed<float>(a, stream);
    case NPA_DTYPE_F16: return backward_typed<__half>(a, stream);
    default: return backward_typed<__nv_bfloat16>(a, stream);
  }
}

uint64_t layer_norm_timeouts() {
  unsigned long long v = 0;
  if (cudaMemcpyFromSymbol(&v, g_timeouts, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}

}  // namespace npa
