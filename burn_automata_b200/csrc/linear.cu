// linear.cu -- matrix product with bias, activation and residual, and its
// backward pass.
//
//   z = x W^T + b,  y = act(z) + r;  dz = dy act'(z),
//   dx = dz W,  dW = dz^T x,  db = sum over rows of dz.
#include <algorithm>

#include "layers.h"

namespace npa {
namespace {

__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case NPA_ACTIVATION_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays NaN
    case NPA_ACTIVATION_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case NPA_ACTIVATION_GELU_TANH:
      return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    case NPA_ACTIVATION_SILU: return z / (1.0f + expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float activation_slope(float z, int act) {
  switch (act) {
    case NPA_ACTIVATION_RELU: return z <= 0.0f ? 0.0f : 1.0f;
    case NPA_ACTIVATION_GELU:
      return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
             z * 0.39894228040143268f * expf(-0.5f * z * z);
    case NPA_ACTIVATION_GELU_TANH: {
      const float t = tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z));
      return 0.5f * (1.0f + t) +
             0.5f * z * (1.0f - t * t) * 0.79788456080286536f * (1.0f + 0.134145f * z * z);
    }
    case NPA_ACTIVATION_SILU: {
      const float s = 1.0f / (1.0f + expf(-z));
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
}

// One operand of a product: value (i, k) at i * si + k * sk.
struct Operand {
  const void* p;
  int64_t si, sk;
};
struct Product {
  Operand a, b;  // a: [m][k], b: [n][k]
  int64_t m, n, k;
  int64_t k_split;  // k values per grid layer
  float* partials;  // [splits][m][n] when split, else null
  const void* bias;
  const void* residual;
  int64_t residual_stride;
  void* y;
  int64_t y_stride;
  void* z;
  int64_t z_stride;
  int act;
};

template <class T>
__device__ __forceinline__ void finish(const Product& p, int64_t i, int64_t j, float z) {
  if (p.bias) z += to_f32(static_cast<const T*>(p.bias)[j]);
  if (p.z) static_cast<T*>(p.z)[i * p.z_stride + j] = from_f32<T>(z);
  float y = activate(z, p.act);
  if (p.residual) y += to_f32(static_cast<const T*>(p.residual)[i * p.residual_stride + j]);
  static_cast<T*>(p.y)[i * p.y_stride + j] = from_f32<T>(y);
}

template <class T>
__global__ void __launch_bounds__(256) product_kernel(Product p) {
  __shared__ float as[16][65], bs[16][65];
  const int64_t m0 = int64_t(blockIdx.x) * 64, n0 = int64_t(blockIdx.y) * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t kb = blockIdx.z * p.k_split;
  const int64_t ke = kb + p.k_split < p.k ? kb + p.k_split : p.k;
  float acc[4][4] = {};
  for (int64_t k0 = kb; k0 < ke; k0 += 16) {
    for (int e = threadIdx.x; e < 1024; e += 256) {
      // the axis with unit stride runs over neighbouring threads
      const int ka = p.a.sk == 1 ? e & 15 : e >> 6, ia = p.a.sk == 1 ? e >> 4 : e & 63;
      const int kc = p.b.sk == 1 ? e & 15 : e >> 6, ib = p.b.sk == 1 ? e >> 4 : e & 63;
      as[ka][ia] = m0 + ia < p.m && k0 + ka < ke
                       ? to_f32(static_cast<const T*>(p.a.p)[(m0 + ia) * p.a.si + (k0 + ka) * p.a.sk])
                       : 0.0f;
      bs[kc][ib] = n0 + ib < p.n && k0 + kc < ke
                       ? to_f32(static_cast<const T*>(p.b.p)[(n0 + ib) * p.b.si + (k0 + kc) * p.b.sk])
                       : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += as[k][ty + 16 * i] * bs[k][tx + 16 * j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
      if (r >= p.m || c >= p.n) continue;
      if (p.partials)
        p.partials[(blockIdx.z * p.m + r) * p.n + c] = acc[i][j];
      else
        finish<T>(p, r, c, acc[i][j]);
    }
}

// The split product's layers summed in order.
template <class T>
__global__ void __launch_bounds__(256) product_reduce_kernel(Product p, int splits) {
  const int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (e >= p.m * p.n) return;
  float s = 0.0f;
  for (int k = 0; k < splits; ++k) s += p.partials[k * p.m * p.n + e];
  finish<T>(p, e / p.n, e % p.n, s);
}

// dz = dy act'(z) as contiguous rows, and per-block column sums of the
// unrounded dz.
template <class T>
__global__ void __launch_bounds__(256) slope_kernel(const T* dy, int64_t dy_stride, const T* z,
                                                    int64_t z_stride, int64_t rows, int outputs,
                                                    int64_t rows_per_block, int act, T* dz,
                                                    float* partials) {
  const int col = blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= outputs) return;
  const int64_t begin = blockIdx.y * rows_per_block;
  const int64_t end = begin + rows_per_block < rows ? begin + rows_per_block : rows;
  float s = 0.0f;
  for (int64_t r = begin; r < end; ++r) {
    float d = to_f32(dy[r * dy_stride + col]);
    if (z) d *= activation_slope(to_f32(z[r * z_stride + col]), act);
    s += d;
    if (dz) dz[r * outputs + col] = from_f32<T>(d);
  }
  partials[int64_t(blockIdx.y) * outputs + col] = s;
}
template <class T>
__global__ void __launch_bounds__(256) bias_reduce_kernel(const float* partials, int count,
                                                          int outputs, T* dbias) {
  const int col = blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= outputs) return;
  float s = 0.0f;
  for (int p = 0; p < count; ++p) s += partials[int64_t(p) * outputs + col];
  dbias[col] = from_f32<T>(s);
}

constexpr int kBiasSplits = 256;

int weight_splits(int64_t rows, int inputs, int outputs) {
  const int64_t tiles = int64_t((inputs + 63) / 64) * ((outputs + 63) / 64);
  const int64_t want = std::max<int64_t>(1, 592 / tiles);
  return int(std::max<int64_t>(1, std::min<int64_t>(want, rows / 256)));
}

struct BackwardCarve {
  void* dz;
  float* bias_partials;
  float* weight_partials;
  size_t bytes;
};
BackwardCarve carve_backward(void* ws, int dtype, int activation, int64_t rows, int inputs,
                             int outputs) {
  Carve c(ws, 0);
  BackwardCarve b{};
  b.dz = activation != NPA_ACTIVATION_IDENTITY
             ? static_cast<void*>(c.take<char>(size_t(rows) * outputs * dtype_bytes(dtype)))
             : nullptr;
  b.bias_partials = c.take<float>(size_t(kBiasSplits) * outputs);
  const int splits = weight_splits(rows, inputs, outputs);
  b.weight_partials = splits > 1 ? c.take<float>(size_t(splits) * inputs * outputs) : nullptr;
  b.bytes = c.used;
  return b;
}

template <class T>
npa_status run_product(const Product& p, int splits, cudaStream_t s) {
  const dim3 grid(unsigned((p.m + 63) / 64), unsigned((p.n + 63) / 64), unsigned(splits));
  product_kernel<T><<<grid, 256, 0, s>>>(p);
  NPA_TRY(after_launch("product_kernel"));
  if (!p.partials) return NPA_OK;
  product_reduce_kernel<T><<<grid_for(uint64_t(p.m * p.n), 256), 256, 0, s>>>(p, splits);
  return after_launch("product_reduce_kernel");
}

template <class T>
npa_status forward_typed(const LinearArgs& a, cudaStream_t s) {
  Product p{};
  p.a = {a.x, a.x_stride, 1};
  p.b = {a.weight, a.weight_stride, 1};
  p.m = a.rows;
  p.n = a.outputs;
  p.k = p.k_split = a.inputs;
  p.bias = a.bias;
  p.residual = a.residual;
  p.residual_stride = a.residual_stride;
  p.y = a.y;
  p.y_stride = a.y_stride;
  p.z = a.z;
  p.z_stride = a.z_stride;
  p.act = a.activation;
  return run_product<T>(p, 1, s);
}

template <class T>
npa_status backward_typed(const LinearBackwardArgs& a, const BackwardCarve& ws, cudaStream_t s) {
  if (a.rows == 0) {
    if (a.dweight)
      NPA_CUDA(cudaMemsetAsync(a.dweight, 0, size_t(a.inputs) * a.outputs * sizeof(T), s),
               "cudaMemsetAsync");
    if (a.dbias)
      NPA_CUDA(cudaMemsetAsync(a.dbias, 0, size_t(a.outputs) * sizeof(T), s), "cudaMemsetAsync");
    return NPA_OK;
  }
  const T* dz = static_cast<const T*>(a.dy);
  int64_t dz_stride = a.dy_stride;
  if (a.dbias || (a.z && (a.dx || a.dweight))) {
    int parts = int(std::min<int64_t>(kBiasSplits, (a.rows + 63) / 64));
    const int64_t per = (a.rows + parts - 1) / parts;
    parts = int((a.rows + per - 1) / per);
    slope_kernel<T><<<dim3(unsigned((a.outputs + 255) / 256), unsigned(parts)), 256, 0, s>>>(
        dz, dz_stride, static_cast<const T*>(a.z), a.z_stride, a.rows, a.outputs, per,
        a.activation, static_cast<T*>(a.z ? ws.dz : nullptr), ws.bias_partials);
    NPA_TRY(after_launch("slope_kernel"));
    if (a.dbias) {
      bias_reduce_kernel<T><<<grid_for(a.outputs, 256), 256, 0, s>>>(
          ws.bias_partials, parts, a.outputs, static_cast<T*>(a.dbias));
      NPA_TRY(after_launch("bias_reduce_kernel"));
    }
    if (a.z) {
      dz = static_cast<const T*>(ws.dz);
      dz_stride = a.outputs;
    }
  }
  if (a.dx) {
    Product p{};
    p.a = {dz, dz_stride, 1};
    p.b = {a.weight, 1, a.weight_stride};
    p.m = a.rows;
    p.n = a.inputs;
    p.k = p.k_split = a.outputs;
    p.y = a.dx;
    p.y_stride = a.dx_stride;
    NPA_TRY(run_product<T>(p, 1, s));
  }
  if (a.dweight) {
    Product p{};
    p.a = {dz, 1, dz_stride};
    p.b = {a.x, 1, a.x_stride};
    p.m = a.outputs;
    p.n = a.inputs;
    p.k = a.rows;
    int splits = weight_splits(a.rows, a.inputs, a.outputs);
    p.k_split = (a.rows + splits - 1) / splits;
    splits = int((a.rows + p.k_split - 1) / p.k_split);
    p.partials = splits > 1 ? ws.weight_partials : nullptr;
    p.y = a.dweight;
    p.y_stride = a.inputs;
    NPA_TRY(run_product<T>(p, splits, s));
  }
  return NPA_OK;
}

}  // namespace

size_t linear_workspace(int, int64_t, int, int) { return 0; }

npa_status launch_linear(int dtype, const LinearArgs& a, void*, cudaStream_t stream) {
  switch (dtype) {
    case NPA_DTYPE_F32: return forward_typed<float>(a, stream);
    case NPA_DTYPE_F16: return forward_typed<__half>(a, stream);
    default: return forward_typed<__nv_bfloat16>(a, stream);
  }
}

size_t linear_backward_workspace(int dtype, int activation, int64_t rows, int inputs, int outputs) {
  if (rows == 0) return 0;
  return carve_backward(nullptr, dtype, activation, rows, inputs, outputs).bytes;
}

npa_status launch_linear_backward(int dtype, const LinearBackwardArgs& a, void* workspace,
                                  cudaStream_t stream) {
  const BackwardCarve ws =
      carve_backward(workspace, dtype, a.activation, a.rows, a.inputs, a.outputs);
  switch (dtype) {
    case NPA_DTYPE_F32: return backward_typed<float>(a, ws, stream);
    case NPA_DTYPE_F16: return backward_typed<__half>(a, ws, stream);
    default: return backward_typed<__nv_bfloat16>(a, ws, stream);
  }
}

}  // namespace npa
