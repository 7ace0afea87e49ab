// capi_layers.cu -- the extern "C" boundary of the normalised-linear operators
// (include/npa_b200.h): every argument is checked before the first CUDA call.
#include <cmath>
#include <new>

#include "host_state.h"
#include "layers.h"

using namespace npa;

namespace {

// Row counts and widths index with 32-bit tile coordinates; element offsets
// are 64-bit.
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024;
constexpr int64_t kMaxDims = int64_t(1) << 24;

npa_status check_dtype(int32_t dtype) {
  if (dtype != NPA_DTYPE_F32 && dtype != NPA_DTYPE_F16 && dtype != NPA_DTYPE_BF16)
    return fail(NPA_ERR_INVALID_ARGUMENT, "unknown dtype " + std::to_string(dtype));
  return NPA_OK;
}

npa_status check_activation(int32_t activation) {
  if (activation < NPA_ACTIVATION_IDENTITY || activation > NPA_ACTIVATION_SILU)
    return fail(NPA_ERR_INVALID_ARGUMENT, "unknown activation " + std::to_string(activation));
  return NPA_OK;
}

npa_status check_size(const char* name, int64_t value, int64_t least, int64_t most) {
  if (value < least)
    return fail(NPA_ERR_INVALID_ARGUMENT, std::string(name) + " must be >= " +
                                              std::to_string(least) + ", got " +
                                              std::to_string(value));
  if (value > most)
    return fail(NPA_ERR_UNSUPPORTED, std::string(name) + " " + std::to_string(value) +
                                         " is above " + std::to_string(most));
  return NPA_OK;
}

// A buffer of `rows` rows: present unless optional or empty, aligned to its
// values, rows that do not overlap.
npa_status check_buffer(const char* name, const void* p, int64_t stride, int64_t rows,
                        int64_t width, size_t size, bool required) {
  if (!p) {
    if (required && rows > 0)
      return fail(NPA_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
    return NPA_OK;
  }
  if (reinterpret_cast<uintptr_t>(p) % size)
    return fail(NPA_ERR_INVALID_ARGUMENT, std::string(name) + " is not aligned to its values");
  if (stride < width)
    return fail(NPA_ERR_INVALID_ARGUMENT, std::string(name) + " stride " + std::to_string(stride) +
                                              " is below the row width " + std::to_string(width));
  if (stride > (int64_t(1) << 40) / (rows > 1 ? rows : 1))
    return fail(NPA_ERR_UNSUPPORTED, std::string(name) + " spans more than 2^40 values");
  return NPA_OK;
}

npa_status check_workspace(const void* workspace, size_t given, size_t needed) {
  if (needed == 0) return NPA_OK;
  if (given < needed)
    return fail(NPA_ERR_INVALID_ARGUMENT, "workspace too small: " + std::to_string(given) +
                                              " bytes, " + std::to_string(needed) + " needed");
  if (!workspace) return fail(NPA_ERR_INVALID_ARGUMENT, "workspace is null");
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(NPA_ERR_INVALID_ARGUMENT, "workspace is not 256-byte aligned");
  return NPA_OK;
}

// Nothing thrown (an allocation of a message, say) leaves a C entry point.
template <class F>
npa_status guarded(F&& body) {
  try {
    return body();
  } catch (const std::bad_alloc&) {
    return NPA_ERR_OUT_OF_MEMORY;
  } catch (...) {
    return NPA_ERR_INVALID_ARGUMENT;
  }
}

Watermarks g_layer_timeouts_seen;

npa_status check_norm_shape(int32_t dtype, int64_t rows, int64_t dims) {
  NPA_TRY(check_dtype(dtype));
  NPA_TRY(check_size("rows", rows, 0, kMaxRows));
  return check_size("dims", dims, 1, kMaxDims);
}

npa_status check_linear_shape(int32_t dtype, int64_t rows, int64_t inputs, int64_t outputs) {
  NPA_TRY(check_dtype(dtype));
  NPA_TRY(check_size("rows", rows, 0, kMaxRows));
  NPA_TRY(check_size("inputs", inputs, 1, kMaxDims));
  return check_size("outputs", outputs, 1, kMaxDims);
}

}  // namespace

extern "C" {

npa_status npa_dev_layer_norm(int32_t dtype, const void* d_x, int64_t x_stride,
                              const void* d_weight, const void* d_bias, int64_t rows, int64_t dims,
                              float eps, void* d_y, int64_t y_stride, float* d_mean, float* d_rstd,
                              void* stream) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_norm_shape(dtype, rows, dims));
    if (!std::isfinite(eps) || eps <= 0.0f)
      return fail_with(NPA_ERR_INVALID_EPS,
                       "eps must be finite and positive, got " + std::to_string(eps), 0, 0, eps);
    const size_t sz = dtype_bytes(dtype);
    NPA_TRY(check_buffer("x", d_x, x_stride, rows, dims, sz, true));
    NPA_TRY(check_buffer("weight", d_weight, dims, 1, dims, sz, false));
    NPA_TRY(check_buffer("bias", d_bias, dims, 1, dims, sz, false));
    NPA_TRY(check_buffer("y", d_y, y_stride, rows, dims, sz, true));
    NPA_TRY(check_buffer("mean", d_mean, 1, rows, 1, 4, false));
    NPA_TRY(check_buffer("rstd", d_rstd, 1, rows, 1, 4, false));
    if (rows == 0) return NPA_OK;
    const LayerNormArgs a{d_x,      x_stride, d_weight, d_bias, rows,  int(dims),
                          eps,      d_y,      y_stride, d_mean, d_rstd};
    return launch_layer_norm(dtype, a, static_cast<cudaStream_t>(stream));
  });
}

npa_status npa_dev_layer_norm_backward_workspace_size(int32_t dtype, int64_t rows, int64_t dims,
                                                      size_t* bytes) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_norm_shape(dtype, rows, dims));
    if (!bytes) return fail(NPA_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = layer_norm_backward_workspace(rows, int(dims));
    return NPA_OK;
  });
}

npa_status npa_dev_layer_norm_backward(int32_t dtype, const void* d_dy, int64_t dy_stride,
                                       const void* d_x, int64_t x_stride, const float* d_mean,
                                       const float* d_rstd, const void* d_weight,
                                       const void* d_residual_gradient,
                                       int64_t residual_gradient_stride, int64_t rows, int64_t dims,
                                       void* d_dx, int64_t dx_stride, void* d_dweight,
                                       void* d_dbias, void* d_workspace, size_t workspace_bytes,
                                       void* stream) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_norm_shape(dtype, rows, dims));
    const size_t sz = dtype_bytes(dtype);
    NPA_TRY(check_buffer("dy", d_dy, dy_stride, rows, dims, sz, true));
    NPA_TRY(check_buffer("x", d_x, x_stride, rows, dims, sz, true));
    NPA_TRY(check_buffer("mean", d_mean, 1, rows, 1, 4, true));
    NPA_TRY(check_buffer("rstd", d_rstd, 1, rows, 1, 4, true));
    NPA_TRY(check_buffer("weight", d_weight, dims, 1, dims, sz, false));
    NPA_TRY(check_buffer("residual_gradient", d_residual_gradient, residual_gradient_stride, rows,
                         dims, sz, false));
    NPA_TRY(check_buffer("dx", d_dx, dx_stride, rows, dims, sz, false));
    NPA_TRY(check_buffer("dweight", d_dweight, dims, 1, dims, sz, false));
    NPA_TRY(check_buffer("dbias", d_dbias, dims, 1, dims, sz, false));
    if (d_residual_gradient && !d_dx && rows > 0)
      return fail(NPA_ERR_INVALID_ARGUMENT, "residual_gradient is added to dx, which is null");
    if (d_dweight || d_dbias)
      NPA_TRY(check_workspace(d_workspace, workspace_bytes,
                              layer_norm_backward_workspace(rows, int(dims))));
    const LayerNormBackwardArgs a{d_dy,   dy_stride, d_x,       x_stride,  d_mean,
                                  d_rstd, d_weight,  d_residual_gradient, residual_gradient_stride,
                                  rows,   int(dims), d_dx,      dx_stride, d_dweight,
                                  d_dbias, static_cast<float*>(d_workspace)};
    return launch_layer_norm_backward(dtype, a, static_cast<cudaStream_t>(stream));
  });
}

npa_status npa_dev_linear_workspace_size(int32_t dtype, int64_t rows, int64_t inputs,
                                         int64_t outputs, size_t* bytes) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_linear_shape(dtype, rows, inputs, outputs));
    if (!bytes) return fail(NPA_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = linear_workspace(dtype, rows, int(inputs), int(outputs));
    return NPA_OK;
  });
}

npa_status npa_dev_linear(int32_t dtype, int32_t activation, const void* d_x, int64_t x_stride,
                          const void* d_weight, int64_t weight_stride, const void* d_bias,
                          const void* d_residual, int64_t residual_stride, int64_t rows,
                          int64_t inputs, int64_t outputs, void* d_y, int64_t y_stride,
                          void* d_pre_activation, int64_t pre_activation_stride,
                          void* d_workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_linear_shape(dtype, rows, inputs, outputs));
    NPA_TRY(check_activation(activation));
    const size_t sz = dtype_bytes(dtype);
    NPA_TRY(check_buffer("x", d_x, x_stride, rows, inputs, sz, true));
    NPA_TRY(check_buffer("weight", d_weight, weight_stride, rows > 0 ? outputs : 0, inputs, sz,
                         true));
    NPA_TRY(check_buffer("bias", d_bias, outputs, 1, outputs, sz, false));
    NPA_TRY(check_buffer("residual", d_residual, residual_stride, rows, outputs, sz, false));
    NPA_TRY(check_buffer("y", d_y, y_stride, rows, outputs, sz, true));
    NPA_TRY(check_buffer("pre_activation", d_pre_activation, pre_activation_stride, rows, outputs,
                         sz, false));
    NPA_TRY(check_workspace(d_workspace, workspace_bytes,
                            linear_workspace(dtype, rows, int(inputs), int(outputs))));
    if (rows == 0) return NPA_OK;
    const LinearArgs a{d_x,  x_stride,    d_weight,     weight_stride, d_bias,
                       d_residual, residual_stride, rows, int(inputs), int(outputs),
                       d_y,  y_stride,    d_pre_activation, pre_activation_stride, activation};
    return launch_linear(dtype, a, d_workspace, static_cast<cudaStream_t>(stream));
  });
}

npa_status npa_dev_linear_backward_workspace_size(int32_t dtype, int32_t activation, int64_t rows,
                                                  int64_t inputs, int64_t outputs, size_t* bytes) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_linear_shape(dtype, rows, inputs, outputs));
    NPA_TRY(check_activation(activation));
    if (!bytes) return fail(NPA_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = linear_backward_workspace(dtype, activation, rows, int(inputs), int(outputs));
    return NPA_OK;
  });
}

npa_status npa_dev_linear_backward(int32_t dtype, int32_t activation, const void* d_dy,
                                   int64_t dy_stride, const void* d_x, int64_t x_stride,
                                   const void* d_weight, int64_t weight_stride,
                                   const void* d_pre_activation, int64_t pre_activation_stride,
                                   int64_t rows, int64_t inputs, int64_t outputs, void* d_dx,
                                   int64_t dx_stride, void* d_dweight, void* d_dbias,
                                   void* d_workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> npa_status {
    NPA_TRY(check_linear_shape(dtype, rows, inputs, outputs));
    NPA_TRY(check_activation(activation));
    const size_t sz = dtype_bytes(dtype);
    const bool any = d_dx || d_dweight || d_dbias;
    const bool slope = activation != NPA_ACTIVATION_IDENTITY;
    NPA_TRY(check_buffer("dy", d_dy, dy_stride, rows, outputs, sz, any));
    NPA_TRY(check_buffer("x", d_x, x_stride, rows, inputs, sz, d_dweight != nullptr));
    NPA_TRY(check_buffer("weight", d_weight, weight_stride, rows > 0 ? outputs : 0, inputs, sz,
                         d_dx != nullptr));
    if (slope)
      NPA_TRY(check_buffer("pre_activation", d_pre_activation, pre_activation_stride, rows,
                           outputs, sz, any));
    NPA_TRY(check_buffer("dx", d_dx, dx_stride, rows, inputs, sz, false));
    NPA_TRY(check_buffer("dweight", d_dweight, inputs, outputs, inputs, sz, false));
    NPA_TRY(check_buffer("dbias", d_dbias, outputs, 1, outputs, sz, false));
    NPA_TRY(check_workspace(
        d_workspace, workspace_bytes,
        linear_backward_workspace(dtype, activation, rows, int(inputs), int(outputs))));
    const LinearBackwardArgs a{d_dy, dy_stride, d_x, x_stride, d_weight, weight_stride,
                               slope ? d_pre_activation : nullptr, pre_activation_stride,
                               rows, int(inputs), int(outputs), d_dx, dx_stride, d_dweight,
                               d_dbias, activation};
    return launch_linear_backward(dtype, a, d_workspace, static_cast<cudaStream_t>(stream));
  });
}

npa_status npa_dev_check_layer_waits(void* stream) {
  return guarded([&]() -> npa_status {
    int dev = 0;
    NPA_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
    NPA_CUDA(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)), "cudaStreamSynchronize");
    if (!g_layer_timeouts_seen.grown(dev, layer_norm_timeouts() + linear_timeouts())) return NPA_OK;
    return fail(NPA_ERR_TIMEOUT,
                "a bounded wait of the layer norm or linear kernels gave up; outputs of calls since the "
                "last check may be unwritten");
  });
}

}  // extern "C"
