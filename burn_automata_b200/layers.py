"""Layer norm and the linear layer with its epilogue, forward and backward.

The layers of a per-particle update block on torch CUDA tensors (float32,
float16 or bfloat16), enqueued on the current torch stream of the tensors'
device through the npa_dev_* entry points.  They have no counterpart in the
reference, whose update MLP is a fixed relu pair of at most 256 hidden units
(NpaModel); they take any width.

Inputs are [..., width]; leading axes are rows.  A 2-D column range of a wider
tensor is read in place; other layouts are copied to rows first.  A caller that
hands over tensors allocated on another stream orders the streams itself, as
for any torch operation.  Gradients are explicit calls (as training.py's);
autograd does not see them.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass
from typing import Optional

from . import _lib
from .config import Activation, InvalidArgument


@dataclass
class LayerNormOutput:
    """y as the input's shape; mean and rstd are float32 [rows...]."""

    y: "torch.Tensor"
    mean: "torch.Tensor"
    rstd: "torch.Tensor"


@dataclass
class LayerNormGradients:
    """Gradients of layer_norm's x, weight and bias (None where not needed)."""

    x: Optional["torch.Tensor"]
    weight: Optional["torch.Tensor"]
    bias: Optional["torch.Tensor"]


@dataclass
class LinearOutput:
    """y and, when it was asked for, the pre-activation z."""

    y: "torch.Tensor"
    pre_activation: Optional["torch.Tensor"]


@dataclass
class LinearGradients:
    """Gradients of linear's x, weight and bias (None where not needed).  The
    residual's gradient is dy itself."""

    x: Optional["torch.Tensor"]
    weight: Optional["torch.Tensor"]
    bias: Optional["torch.Tensor"]


_torch = None
_dtypes = {}
_raw_stream = None


def _t():
    global _torch, _raw_stream
    if _torch is None:
        import torch

        _dtypes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        # a stream object costs microseconds; the handle alone does not
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _torch = torch
    return _torch


def _dtype(x, name: str) -> int:
    """The C ABI's storage type of a CUDA tensor."""
    torch = _torch or _t()
    if not isinstance(x, torch.Tensor):
        raise InvalidArgument(f"{name} must be a torch tensor")
    code = _dtypes.get(x.dtype)
    if code is None:
        raise InvalidArgument(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise InvalidArgument(f"{name} must be a CUDA tensor")
    if x.dim() < 1:
        raise InvalidArgument(f"{name} needs at least one axis")
    return code


def _like(t, x, name: str):
    if not isinstance(t, _torch.Tensor):
        raise InvalidArgument(f"{name} must be a torch tensor")
    if t.dtype != x.dtype or t.device != x.device:
        raise InvalidArgument(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")


def _rows(t):
    """(tensor, row stride) with unit stride inside rows: the tensor itself for
    a contiguous tensor or a 2-D column range, else a contiguous copy."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t, t.stride(0)
    return t.contiguous(), t.shape[-1]


def _aligned_rows(t, work: int, reuse: int):
    """As _rows for a product's operand: one whose rows do not all start on 16
    bytes (by its stride or by its address), but would in a copy of its own, is
    copied where that pays.  `work` is the product's multiplications, `reuse` how
    many of them a value takes part in.  16 bits: TMA reads aligned rows only, and
    the loader warps that read others lose more than a copy takes from 2^30 on (x
    one value off, forward, us without and with it: 16384 x 512 -> 2048 262 and 46,
    300000 x 64 -> 128 64 and 50; 2^29: 16384 x 256 -> 128 15 and 24).  f32 goes
    through them either way and gains on values that are read often (65536 x 128 ->
    1024 187 and 142; 65536 x 1024 -> 128 194 and 221)."""
    t, stride = _rows(t)
    if work < 1 << 30:
        return t, stride
    size = t.element_size()
    if ((t.data_ptr() % 16 or (stride * size) % 16 and t.shape[0] > 1)
            and t.shape[-1] * size % 16 == 0 and (size == 2 or reuse >= 384)):
        return t.clone(memory_format=_t().contiguous_format), t.shape[-1]
    return t, stride


def _matrix(t, x, shape, name: str):
    _like(t, x, name)
    if t.shape != shape:
        raise InvalidArgument(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return _rows(t)


def _vector(t, x, size: int, name: str):
    if t is None:
        return None
    _like(t, x, name)
    if t.dim() != 1 or t.shape[0] != size:
        raise InvalidArgument(f"{name} has shape {tuple(t.shape)}, expected ({size},)")
    return t if t.is_contiguous() else t.contiguous()


def _statistic(t, x, name: str):
    if not isinstance(t, _torch.Tensor) or t.dtype != _torch.float32 or t.device != x.device:
        raise InvalidArgument(f"{name} must be a float32 tensor on {x.device}")
    if t.shape != x.shape[:-1]:
        raise InvalidArgument(f"{name} has shape {tuple(t.shape)}, expected "
                              f"{tuple(x.shape[:-1])}")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _needs(needs):
    want = set(needs)
    if not want <= {"x", "weight", "bias"}:
        raise InvalidArgument(f"needs may name x, weight and bias, got {sorted(want)}")
    return want


def _call(entry, device, args, name: str) -> None:
    """entry(*args, stream) on the device's current stream."""
    index = device.index
    if index == _torch.cuda.current_device():
        status = entry(*args, _raw_stream(index))
    else:
        with _torch.cuda.device(index):
            status = entry(*args, _raw_stream(index))
    if status:
        _lib.check(status, name)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(query: str, *args) -> int:
    """The workspace size that the C ABI's query gives for these sizes."""
    need = ctypes.c_size_t(0)
    _lib.check(getattr(_lib.lib(), query)(*args, ctypes.byref(need)), query)
    return need.value


def _workspace(x, query: str, *args):
    """(pointer's owner or None, bytes) of one call's workspace."""
    need = _workspace_bytes(query, *args)
    return (x.new_empty(need, dtype=_torch.uint8), need) if need else (None, 0)


def _outputs_like(x, shape):
    """An uninitialised contiguous tensor of x's type."""
    if x.shape == shape and x.is_contiguous():
        return _torch.empty_like(x)
    return x.new_empty(shape)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5) -> LayerNormOutput:
    """(x - mean) * rstd * weight + bias over the last axis, with the mean and
    rstd that layer_norm_backward takes."""
    code = _dtype(x, "x")
    torch = _torch
    dims = x.shape[-1]
    w, b = _vector(weight, x, dims, "weight"), _vector(bias, x, dims, "bias")
    xr, xs = _rows(x)
    y = _outputs_like(x, x.shape)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _call(_lib.lib().npa_dev_layer_norm, x.device,
          (code, xr.data_ptr(), xs, _ptr(w), _ptr(b), mean.numel(), dims, float(eps),
           y.data_ptr(), dims, mean.data_ptr(), rstd.data_ptr()), "layer_norm")
    return LayerNormOutput(y, mean, rstd)


def layer_norm_backward(dy, x, mean, rstd, weight=None, residual_gradient=None,
                        needs=None) -> LayerNormGradients:
    """The gradients of layer_norm given dy and its saved statistics.
    residual_gradient, the gradient that reaches x over a skip connection, is
    added to x's on the way.  `needs` names the gradients to compute: x,
    weight and bias by default, x alone when there is no weight."""
    code = _dtype(x, "x")
    dims = x.shape[-1]
    want = _needs(needs if needs is not None else
                  (("x", "weight", "bias") if weight is not None else ("x",)))
    w = _vector(weight, x, dims, "weight")
    dyr, dys = _matrix(dy, x, x.shape, "dy")
    xr, xs = _rows(x)
    m, r = _statistic(mean, x, "mean"), _statistic(rstd, x, "rstd")
    rr, rs = (None, 0) if residual_gradient is None else _matrix(
        residual_gradient, x, x.shape, "residual_gradient")
    if rr is not None and "x" not in want:
        raise InvalidArgument("residual_gradient is added to x's gradient, which is not needed")
    dx = _outputs_like(x, x.shape) if "x" in want else None
    dw = x.new_empty(dims) if "weight" in want else None
    db = x.new_empty(dims) if "bias" in want else None
    rows = m.numel()
    L = _lib.lib()
    ws, ws_bytes = None, 0
    if dw is not None or db is not None:
        ws, ws_bytes = _workspace(x, "npa_dev_layer_norm_backward_workspace_size", code, rows,
                                  dims)
    _call(L.npa_dev_layer_norm_backward, x.device,
          (code, dyr.data_ptr(), dys, xr.data_ptr(), xs, m.data_ptr(), r.data_ptr(), _ptr(w),
           _ptr(rr), rs, rows, dims, _ptr(dx), dims, _ptr(dw), _ptr(db), _ptr(ws), ws_bytes),
          "layer_norm_backward")
    return LayerNormGradients(dx, dw, db)


def check_layer_waits(device=None) -> None:
    """Waits for the device's current stream and raises DeviceTimeout if a bounded
    wait of the kernels behind this module's calls has given up on the device
    since the last such check: the calls return before their kernels run, and a
    kernel that gives up leaves outputs unwritten.  Once for a training step or a
    batch of requests."""
    torch = _torch or _t()
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    with torch.cuda.device(index):
        status = _lib.lib().npa_dev_check_layer_waits(
            _raw_stream(torch.cuda.current_device()))
    _lib.check(status, "check_layer_waits")


def _activation(activation) -> int:
    if type(activation) is not Activation:
        try:
            activation = Activation(activation)
        except ValueError:
            raise InvalidArgument(f"unknown activation {activation!r}") from None
    return int(activation)


def _layer_shape(x, weight):
    if not isinstance(weight, _t().Tensor) or weight.dim() != 2:
        raise InvalidArgument("weight must be a 2-D tensor [outputs, inputs]")
    if weight.shape[1] != x.shape[-1]:
        raise InvalidArgument(f"weight has {weight.shape[1]} inputs, x has {x.shape[-1]}")
    return weight.shape[1], weight.shape[0]


def linear(x, weight, bias=None, residual=None, activation: Activation = Activation.Identity,
           save_pre_activation: bool = False) -> LinearOutput:
    """activation(x weight^T + bias) + residual, weight [outputs, inputs].
    save_pre_activation also returns z = x weight^T + bias, which
    linear_backward reads for every activation but the identity."""
    code, act = _dtype(x, "x"), _activation(activation)
    torch = _torch
    inputs, outputs = _layer_shape(x, weight)
    out_shape = x.shape[:-1] + (outputs,)
    _like(weight, x, "weight")
    rows = x.numel() // inputs if inputs else 0
    work = rows * inputs * outputs
    wr, wstride = _aligned_rows(weight, work, rows)
    b = _vector(bias, x, outputs, "bias")
    rr, rs = (None, 0) if residual is None else _matrix(residual, x, out_shape, "residual")
    xr, xs = _aligned_rows(x, work, outputs)
    y = _outputs_like(x, out_shape)
    z = torch.empty_like(y) if save_pre_activation else None
    L = _lib.lib()
    ws, ws_bytes = _workspace(x, "npa_dev_linear_workspace_size", code, rows, inputs, outputs)
    _call(L.npa_dev_linear, x.device,
          (code, act, xr.data_ptr(), xs, wr.data_ptr(), wstride, _ptr(b), _ptr(rr), rs,
           rows, inputs, outputs, y.data_ptr(), outputs, _ptr(z), outputs, _ptr(ws), ws_bytes),
          "linear")
    return LinearOutput(y, z)


def linear_backward(dy, x, weight, pre_activation=None,
                    activation: Activation = Activation.Identity,
                    needs=("x", "weight", "bias")) -> LinearGradients:
    """The gradients of linear given dy and (for every activation but the
    identity) its saved pre-activation.  `needs` names the gradients to
    compute."""
    code, act = _dtype(x, "x"), _activation(activation)
    inputs, outputs = _layer_shape(x, weight)
    out_shape = x.shape[:-1] + (outputs,)
    want = _needs(needs)
    _like(weight, x, "weight")
    rows = x.numel() // inputs if inputs else 0
    work = rows * inputs * outputs
    wr, wstride = _aligned_rows(weight, work, rows)
    dyr, dys = _matrix(dy, x, out_shape, "dy")
    zr, zs = None, 0
    if act != Activation.Identity:
        if pre_activation is None:
            raise InvalidArgument("this activation's gradient needs pre_activation")
        zr, zs = _matrix(pre_activation, x, out_shape, "pre_activation")
    else:
        # dy itself is the products' operand; with an activation a pass makes dz of it
        dyr, dys = _aligned_rows(dyr, work, inputs)
    xr, xs = _aligned_rows(x, work, outputs)
    dx = _outputs_like(x, x.shape) if "x" in want else None
    dw = _outputs_like(weight, weight.shape) if "weight" in want else None
    db = x.new_empty(outputs) if "bias" in want else None
    L = _lib.lib()
    ws, ws_bytes = _workspace(x, "npa_dev_linear_backward_workspace_size", code, act, rows,
                              inputs, outputs)
    _call(L.npa_dev_linear_backward, x.device,
          (code, act, dyr.data_ptr(), dys, xr.data_ptr(), xs, wr.data_ptr(), wstride,
           _ptr(zr), zs, rows, inputs, outputs, _ptr(dx), inputs, _ptr(dw), _ptr(db), _ptr(ws),
           ws_bytes), "linear_backward")
    return LinearGradients(dx, dw, db)
