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
#include <algorithm>

#include "layers.h"

namespace npa {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarpRowThreads = 256;  // threads per block where a warp or less has a row

// Sums `a` and `b` over the row's threads.  WARP: tpr lanes (a power of two)
// have a row; else the whole block, through shared memory, whose two halves
// alternate so that one barrier per sum is enough.
struct RowSum {
  float* buf;  // [2][64], block rows only
  int phase = 0;
};
template <bool BLOCK>
__device__ __forceinline__ void row_sum2(RowSum& rs, int tpr, float& a, float& b) {
  for (int o = (BLOCK ? 32 : tpr) >> 1; o > 0; o >>= 1) {
    a += __shfl_xor_sync(kFull, a, o);
    b += __shfl_xor_sync(kFull, b, o);
  }
  if (BLOCK) {
    float* s = rs.buf + rs.phase * 64;
    rs.phase ^= 1;
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      s[warp] = a;
      s[32 + warp] = b;
    }
    __syncthreads();
    a = b = 0.0f;
    for (int w = 0; w < warps; ++w) {
      a += s[w];
      b += s[32 + w];
    }
  }
}
template <bool BLOCK>
__device__ __forceinline__ float row_sum(RowSum& rs, int tpr, float a) {
  for (int o = (BLOCK ? 32 : tpr) >> 1; o > 0; o >>= 1) a += __shfl_xor_sync(kFull, a, o);
  if (BLOCK) {
    float* s = rs.buf + rs.phase * 64;
    rs.phase ^= 1;
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) s[warp] = a;
    __syncthreads();
    a = 0.0f;
    for (int w = 0; w < warps; ++w) a += s[w];
  }
  return a;
}

// Thread `lane` of a row's `tpr` threads has the vectors lane, lane + tpr, ...
// of VEC values, NV of them at most.
template <class T, int VEC, int NV>
__device__ __forceinline__ void load_row(const T* row, int lane, int tpr, int nvec, bool active,
                                         float (&out)[NV * VEC]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int q = lane + k * tpr;
    if (active && q < nvec) {
      const Pack<T, VEC> p = reinterpret_cast<const Pack<T, VEC>*>(row)[q];
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[k * VEC + j] = to_f32(p.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[k * VEC + j] = 0.0f;
    }
  }
}

template <class T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : kWarpRowThreads)
layer_norm_kernel(LayerNormArgs a, int tpr_) {
  __shared__ float sums[128];
  RowSum rs{sums};
  const int tpr = BLOCK ? int(blockDim.x) : tpr_;
  const int lane = BLOCK ? int(threadIdx.x) : int(threadIdx.x) & (tpr - 1);
  const int per_block = BLOCK ? 1 : int(blockDim.x) / tpr;
  const int in_block = BLOCK ? 0 : int(threadIdx.x) / tpr;
  const int nvec = a.dims / VEC;
  const float inv_n = 1.0f / float(a.dims);
  const T* const w = static_cast<const T*>(a.weight);
  const T* const b = static_cast<const T*>(a.bias);
  for (int64_t base = int64_t(blockIdx.x) * per_block; base < a.rows;
       base += int64_t(gridDim.x) * per_block) {
    const int64_t row = base + in_block;
    const bool active = row < a.rows;
    float x[NV * VEC];
    load_row<T, VEC, NV>(static_cast<const T*>(a.x) + row * a.x_stride, lane, tpr, nvec, active,
                         x);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) s += x[e];
    const float mean = row_sum<BLOCK>(rs, tpr, s) * inv_n;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (lane + k * tpr < nvec) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = x[k * VEC + j] - mean;
          v += d * d;
        }
      }
    const float rstd = 1.0f / sqrtf(row_sum<BLOCK>(rs, tpr, v) * inv_n + a.eps);
    if (!active) continue;
    T* const out = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = lane + k * tpr;
      if (q >= nvec) continue;
      Pack<T, VEC> p, wp, bp;
      if (w) wp = reinterpret_cast<const Pack<T, VEC>*>(w)[q];
      if (b) bp = reinterpret_cast<const Pack<T, VEC>*>(b)[q];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float y = (x[k * VEC + j] - mean) * rstd;
        if (w) y *= to_f32(wp.v[j]);
        if (b) y += to_f32(bp.v[j]);
        p.v[j] = from_f32<T>(y);
      }
      reinterpret_cast<Pack<T, VEC>*>(out)[q] = p;
    }
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

// Rows too long for registers: a block walks the row three times (the second
// and third walks find it in L2).
template <class T>
__global__ void __launch_bounds__(512) layer_norm_long_kernel(LayerNormArgs a) {
  __shared__ float sums[128];
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

// PARAMS: each block leaves its rows' dw and db sums in
// partials[block][2][dims].
template <class T, int VEC, int NV, bool BLOCK, bool PARAMS>
__global__ void __launch_bounds__(BLOCK ? 512 : kWarpRowThreads)
layer_norm_backward_kernel(LayerNormBackwardArgs a, int tpr_) {
  constexpr int E = NV * VEC;
  __shared__ float sums[128];
  extern __shared__ float columns[];  // [2][dims], warp rows with PARAMS only
  RowSum rs{sums};
  const int tpr = BLOCK ? int(blockDim.x) : tpr_;
  const int lane = BLOCK ? int(threadIdx.x) : int(threadIdx.x) & (tpr - 1);
  const int per_block = BLOCK ? 1 : int(blockDim.x) / tpr;
  const int in_block = BLOCK ? 0 : int(threadIdx.x) / tpr;
  const int nvec = a.dims / VEC;
  const float inv_n = 1.0f / float(a.dims);
  const T* const w = static_cast<const T*>(a.weight);
  float dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  for (int64_t base = int64_t(blockIdx.x) * per_block; base < a.rows;
       base += int64_t(gridDim.x) * per_block) {
    const int64_t row = base + in_block;
    const bool active = row < a.rows;
    float xh[E], g[E];
    load_row<T, VEC, NV>(static_cast<const T*>(a.x) + row * a.x_stride, lane, tpr, nvec, active,
                         xh);
    load_row<T, VEC, NV>(static_cast<const T*>(a.dy) + row * a.dy_stride, lane, tpr, nvec, active,
                         g);
    const float mean = active ? a.mean[row] : 0.0f, rstd = active ? a.rstd[row] : 0.0f;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = lane + k * tpr;
      if (!active || q >= nvec) continue;
      Pack<T, VEC> wp;
      if (w) wp = reinterpret_cast<const Pack<T, VEC>*>(w)[q];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = k * VEC + j;
        xh[e] = (xh[e] - mean) * rstd;
        if (PARAMS) {
          dw[e] += g[e] * xh[e];
          db[e] += g[e];
        }
        if (w) g[e] *= to_f32(wp.v[j]);
        s1 += g[e];
        s2 += g[e] * xh[e];
      }
    }
    if (!a.dx) continue;
    row_sum2<BLOCK>(rs, tpr, s1, s2);
    if (!active) continue;
    s1 *= inv_n;
    s2 *= inv_n;
    T* const out = static_cast<T*>(a.dx) + row * a.dx_stride;
    const T* const res =
        a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = lane + k * tpr;
      if (q >= nvec) continue;
      Pack<T, VEC> p, rp;
      if (res) rp = reinterpret_cast<const Pack<T, VEC>*>(res)[q];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = k * VEC + j;
        float d = rstd * (g[e] - s1 - xh[e] * s2);
        if (res) d += to_f32(rp.v[j]);
        p.v[j] = from_f32<T>(d);
      }
      reinterpret_cast<Pack<T, VEC>*>(out)[q] = p;
    }
  }
  if (!PARAMS) return;
  float* const part = a.partials + int64_t(blockIdx.x) * 2 * a.dims;
  if (BLOCK) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = lane + k * tpr;
      if (q >= nvec) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        part[q * VEC + j] = dw[k * VEC + j];
        part[a.dims + q * VEC + j] = db[k * VEC + j];
      }
    }
    return;
  }
  for (int group = 0; group < per_block; ++group) {
    if (group == in_block) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int q = lane + k * tpr;
        if (q >= nvec) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float* const cw = columns + q * VEC + j;
          *cw = group == 0 ? dw[k * VEC + j] : *cw + dw[k * VEC + j];
          cw[a.dims] = group == 0 ? db[k * VEC + j] : cw[a.dims] + db[k * VEC + j];
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.dims; i += blockDim.x) part[i] = columns[i];
}

// Long rows: dx by a block per row in two walks; dw and db by
// column_partials_kernel.
template <class T>
__global__ void __launch_bounds__(512) layer_norm_backward_long_kernel(LayerNormBackwardArgs a) {
  __shared__ float sums[128];
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

// dw and db from the blocks' partial sums: 32 columns per block, whose 8 row
// lanes each add every eighth partial in order and meet in a fixed tree.
template <class T>
__global__ void __launch_bounds__(256) column_reduce_kernel(const float* __restrict__ partials,
                                                            int count, int dims, T* dweight,
                                                            T* dbias) {
  __shared__ float acc[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t col = int64_t(blockIdx.x) * 32 + tx;  // over [2][dims]
  float s = 0.0f;
  if (col < 2 * int64_t(dims))
    for (int p = ty; p < count; p += 8) s += partials[int64_t(p) * 2 * dims + col];
  acc[ty][tx] = s;
  __syncthreads();
  if (ty != 0 || col >= 2 * int64_t(dims)) return;
  s = ((acc[0][tx] + acc[1][tx]) + (acc[2][tx] + acc[3][tx])) +
      ((acc[4][tx] + acc[5][tx]) + (acc[6][tx] + acc[7][tx]));
  T* const out = col < dims ? dweight : dbias;
  if (out) out[col < dims ? col : col - dims] = from_f32<T>(s);
}

// How a row is spread over threads.
struct RowPlan {
  int vec;      // values per access
  int nv;       // accesses per thread (1, 2, 3, 4 or 8); 0: the long kernel
  int tpr;      // threads per row
  bool block;   // the whole block has one row
};

bool aligned(const void* p, int64_t stride, size_t sz, int vec) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (sz * vec) == 0 && stride % vec == 0);
}

// The widest access that every buffer allows, then the fewest threads whose
// registers hold the row: up to `most` values per thread.
RowPlan plan_row(size_t sz, int dims, int widest, int most) {
  RowPlan p{};
  p.vec = widest;
  const int nvec = dims / p.vec;
  const int nv_most = std::min(8, most / p.vec);
  auto round_nv = [](int nv) { return nv <= 4 ? nv : 8; };
  if (nvec <= 32 * nv_most) {
    int tpr = 4;
    // a row's threads: about four accesses each while a warp has enough
    while (tpr < 32 && (nvec + tpr - 1) / tpr > std::min(4, nv_most)) tpr *= 2;
    p.tpr = tpr;
    p.nv = round_nv((nvec + tpr - 1) / tpr);
    return p;
  }
  p.block = true;
  for (int nv : {1, 2, 4, 8}) {
    if (nv > nv_most) break;
    const int threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
    if (threads <= 512) {
      p.nv = nv;
      p.tpr = threads;
      if (threads <= 256) break;
    }
  }
  return p;
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

template <class T, int VEC, int NV, bool PARAMS>
int backward_launch(const LayerNormBackwardArgs& a, const RowPlan& p, cudaStream_t stream) {
  if (p.block) {
    const int64_t grid = std::min<int64_t>(std::min<int64_t>(a.rows, kMaxPartials),
                                             int64_t(sm_count()) * (1024 / p.tpr));
    layer_norm_backward_kernel<T, VEC, NV, true, PARAMS>
        <<<unsigned(grid), p.tpr, 0, stream>>>(a, p.tpr);
    return int(grid);
  }
  const int per_block = kWarpRowThreads / p.tpr;
  const int64_t grid =
      std::min<int64_t>(std::min<int64_t>((a.rows + per_block - 1) / per_block, kMaxPartials),
                        int64_t(sm_count()) * 4);
  const size_t smem = PARAMS ? size_t(a.dims) * 2 * sizeof(float) : 0;
  layer_norm_backward_kernel<T, VEC, NV, false, PARAMS>
      <<<unsigned(grid), kWarpRowThreads, smem, stream>>>(a, p.tpr);
  return int(grid);
}

template <class T, int VEC, bool PARAMS>
int backward_nv(const LayerNormBackwardArgs& a, const RowPlan& p, cudaStream_t s) {
  switch (p.nv) {
    case 1: return backward_launch<T, VEC, 1, PARAMS>(a, p, s);
    case 2: return backward_launch<T, VEC, 2, PARAMS>(a, p, s);
    default: break;
  }
  if constexpr (VEC * 4 <= 16) {
    switch (p.nv) {
      case 3: return backward_launch<T, VEC, 3, PARAMS>(a, p, s);
      case 4: return backward_launch<T, VEC, 4, PARAMS>(a, p, s);
      default: break;
    }
  }
  if constexpr (VEC * 8 <= 16) return backward_launch<T, VEC, 8, PARAMS>(a, p, s);
  return 0;
}

template <class T, bool PARAMS>
int backward_vec(const LayerNormBackwardArgs& a, const RowPlan& p, cudaStream_t s) {
  switch (p.vec) {
    case 1: return backward_nv<T, 1, PARAMS>(a, p, s);
    case 2: return backward_nv<T, 2, PARAMS>(a, p, s);
    case 4: return backward_nv<T, 4, PARAMS>(a, p, s);
    default: break;
  }
  if constexpr (sizeof(T) == 2) return backward_nv<T, 8, PARAMS>(a, p, s);
  return 0;
}

template <class T, int VEC>
void forward_nv(const LayerNormArgs& a, const RowPlan& p, cudaStream_t s) {
  switch (p.nv) {
    case 1: return forward_launch<T, VEC, 1>(a, p, s);
    case 2: return forward_launch<T, VEC, 2>(a, p, s);
    case 3: return forward_launch<T, VEC, 3>(a, p, s);
    case 4: return forward_launch<T, VEC, 4>(a, p, s);
    default: break;
  }
  if constexpr (VEC * 8 <= 32) forward_launch<T, VEC, 8>(a, p, s);
}

template <class T>
npa_status forward_typed(const LayerNormArgs& a, cudaStream_t s) {
  int vec = 16 / int(sizeof(T));
  while (vec > 1 && (a.dims % vec || !aligned(a.x, a.x_stride, sizeof(T), vec) ||
                     !aligned(a.y, a.y_stride, sizeof(T), vec) ||
                     !aligned(a.weight, 0, sizeof(T), vec) || !aligned(a.bias, 0, sizeof(T), vec)))
    vec /= 2;
  const RowPlan p = plan_row(sizeof(T), a.dims, vec, 32);
  if (p.nv == 0) {
    const int64_t grid = std::min<int64_t>(a.rows, int64_t(sm_count()) * 4);
    layer_norm_long_kernel<T><<<unsigned(grid), 512, 0, s>>>(a);
    return after_launch("layer_norm_long_kernel");
  }
  switch (p.vec) {
    case 1: forward_nv<T, 1>(a, p, s); break;
    case 2: forward_nv<T, 2>(a, p, s); break;
    case 4: forward_nv<T, 4>(a, p, s); break;
    default:
      if constexpr (sizeof(T) == 2) forward_nv<T, 8>(a, p, s);
  }
  return after_launch("layer_norm_kernel");
}

template <class T>
npa_status backward_typed(const LayerNormBackwardArgs& a, cudaStream_t s) {
  const bool params = a.dweight || a.dbias;
  int vec = 16 / int(sizeof(T));
  while (vec > 1 &&
         (a.dims % vec || !aligned(a.x, a.x_stride, sizeof(T), vec) ||
          !aligned(a.dy, a.dy_stride, sizeof(T), vec) ||
          !aligned(a.dx, a.dx_stride, sizeof(T), vec) || !aligned(a.weight, 0, sizeof(T), vec) ||
          !aligned(a.residual, a.residual_stride, sizeof(T), vec)))
    vec /= 2;
  const RowPlan p = plan_row(sizeof(T), a.dims, vec, 16);
  int parts = 0;
  if (p.nv == 0) {
    if (a.dx && a.rows > 0) {
      const int64_t grid = std::min<int64_t>(a.rows, int64_t(sm_count()) * 4);
      layer_norm_backward_long_kernel<T><<<unsigned(grid), 512, 0, s>>>(a);
      NPA_TRY(after_launch("layer_norm_backward_long_kernel"));
    }
    if (params && a.rows > 0) {
      parts = int(std::min<int64_t>(a.rows, kLongSplits));
      const int64_t per = (a.rows + parts - 1) / parts;
      parts = int((a.rows + per - 1) / per);
      column_partials_kernel<T><<<dim3(unsigned((a.dims + 255) / 256), unsigned(parts)), 256, 0, s>>>(
          a, per);
      NPA_TRY(after_launch("column_partials_kernel"));
    }
  } else if (a.rows > 0 && (a.dx || params)) {
    parts = params ? backward_vec<T, true>(a, p, s) : backward_vec<T, false>(a, p, s);
    NPA_TRY(after_launch("layer_norm_backward_kernel"));
  }
  if (!params) return NPA_OK;
  column_reduce_kernel<T><<<unsigned((2 * int64_t(a.dims) + 31) / 32), 256, 0, s>>>(
      a.partials, parts, a.dims, static_cast<T*>(a.dweight), static_cast<T*>(a.dbias));
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

}  // namespace npa
