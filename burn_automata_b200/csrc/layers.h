// layers.h -- storage types, activations and launchers of the normalised-linear
// operators (layer_norm.cu, linear.cu; entry points in capi_layers.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "npa_internal.h"

namespace npa {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Results are rounded to the storage type once, to nearest even.
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values to and from f32, the low half first.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  // a bf16 is the upper half of the f32 of the same value
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Two f32 values in a register pair: sm_100 adds, multiplies and fuses pairs in
// one instruction.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 values(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// VEC consecutive values, loaded and stored as one access.
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// A call's kernels follow each other with programmatic dependent launches: each
// lets the next one's blocks in as soon as its own have started, and each waits
// for the one before to end before it touches memory.  What overlaps is the
// launch itself and what a kernel sets up for itself.
__device__ __forceinline__ void let_next_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Launches `kernel` behind the stream's last kernel; `after` = true lets it in
// early (only behind a kernel of the same call, which lets it).
template <class... Params, class... Args>
cudaError_t launch_kernel(bool after, void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                          cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(unsigned(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}

inline size_t dtype_bytes(int dtype) { return dtype == NPA_DTYPE_F32 ? 4 : 2; }

struct LayerNormArgs {
  const void* x;
  int64_t x_stride;
  const void* weight;  // optional
  const void* bias;    // optional
  int64_t rows;
  int dims;
  float eps;
  void* y;
  int64_t y_stride;
  float* mean;  // optional
  float* rstd;  // optional
};
npa_status launch_layer_norm(int dtype, const LayerNormArgs& a, cudaStream_t stream);

struct LayerNormBackwardArgs {
  const void* dy;
  int64_t dy_stride;
  const void* x;
  int64_t x_stride;
  const float* mean;
  const float* rstd;
  const void* weight;    // optional
  const void* residual;  // optional: added to dx
  int64_t residual_stride;
  int64_t rows;
  int dims;
  void* dx;  // optional
  int64_t dx_stride;
  void* dweight;  // optional
  void* dbias;    // optional
  float* partials;
};
// Bounded waits of the layer norm kernels that gave up on the current device.
uint64_t layer_norm_timeouts();
size_t layer_norm_backward_workspace(int64_t rows, int dims);
npa_status launch_layer_norm_backward(int dtype, const LayerNormBackwardArgs& a,
                                      cudaStream_t stream);

struct LinearArgs {
  const void* x;
  int64_t x_stride;
  const void* weight;
  int64_t weight_stride;
  const void* bias;      // optional
  const void* residual;  // optional
  int64_t residual_stride;
  int64_t rows;
  int inputs, outputs;
  void* y;
  int64_t y_stride;
  void* z;  // optional
  int64_t z_stride;
  int activation;
};
// Bounded waits of the product kernels that gave up on the current device.
uint64_t linear_timeouts();
size_t linear_workspace(int dtype, int64_t rows, int inputs, int outputs);
npa_status launch_linear(int dtype, const LinearArgs& a, void* workspace, cudaStream_t stream);

struct LinearBackwardArgs {
  const void* dy;
  int64_t dy_stride;
  const void* x;
  int64_t x_stride;
  const void* weight;
  int64_t weight_stride;
  const void* z;  // null for the identity
  int64_t z_stride;
  int64_t rows;
  int inputs, outputs;
  void* dx;  // optional
  int64_t dx_stride;
  void* dweight;  // optional
  void* dbias;    // optional
  int activation;
};
size_t linear_backward_workspace(int dtype, int activation, int64_t rows, int inputs, int outputs);
npa_status launch_linear_backward(int dtype, const LinearBackwardArgs& a, void* workspace,
                                  cudaStream_t stream);

}  // namespace npa
