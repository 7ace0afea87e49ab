"""A wide per-particle update network built from layers.py's operators.

Where NpaModel's update is one relu pair of at most 256 hidden units in the
reference's f32 order, this one takes any width and float32, float16 or
bfloat16 weights on the tensor cores:

  h_0     = features                                   [rows, F]
  h_(i+1) = h_i + W2 act(W1 norm(h_i) + b1) + b2       (UpdateBlock)
  next    = states + R norm(h_n) + b                   [rows, C]

It has no counterpart in the reference.  Passes are explicit, as training.py's:
forward keeps what backward reads, and gradients come back as lists in
parameters()'s order.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import List

from . import layers
from .config import Activation, InvalidArgument


def _randn(shape, scale, dtype, device, generator):
    import torch

    return (torch.randn(shape, generator=generator, dtype=torch.float32, device=device)
            * scale).to(dtype)


@dataclass
class _Saved:
    """What one block's backward pass reads."""

    x: "torch.Tensor"
    norm: layers.LayerNormOutput
    hidden: layers.LinearOutput


class UpdateBlock:
    """h + W2 act(W1 norm(h) + b1) + b2 over rows of `features` values."""

    def __init__(self, features: int, hidden: int, activation: Activation = Activation.Gelu,
                 dtype=None, device=None, generator=None, eps: float = 1e-5):
        import torch

        if features < 1 or hidden < 1:
            raise InvalidArgument("features and hidden must be >= 1")
        dtype = dtype or torch.bfloat16
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        self.activation = Activation(activation)
        self.eps = float(eps)
        self.norm_weight = torch.ones(features, dtype=dtype, device=device)
        self.norm_bias = torch.zeros(features, dtype=dtype, device=device)
        self.w1 = _randn((hidden, features), (2.0 / features) ** 0.5, dtype, device, generator)
        self.b1 = torch.zeros(hidden, dtype=dtype, device=device)
        # a small second layer: the block starts near the identity
        self.w2 = _randn((features, hidden), 0.1 * (1.0 / hidden) ** 0.5, dtype, device, generator)
        self.b2 = torch.zeros(features, dtype=dtype, device=device)

    def parameters(self) -> List["torch.Tensor"]:
        return [self.norm_weight, self.norm_bias, self.w1, self.b1, self.w2, self.b2]

    def forward(self, x, save: bool = True):
        """(output, what backward reads or None)."""
        norm = layers.layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        hidden = layers.linear(norm.y, self.w1, self.b1, activation=self.activation,
                               save_pre_activation=save)
        out = layers.linear(hidden.y, self.w2, self.b2, residual=x).y
        return out, (_Saved(x, norm, hidden) if save else None)

    def backward(self, dy, saved: _Saved):
        """(gradient of x, gradients in parameters()'s order)."""
        second = layers.linear_backward(dy, saved.hidden.y, self.w2)
        first = layers.linear_backward(second.x, saved.norm.y, self.w1,
                                       saved.hidden.pre_activation, activation=self.activation)
        norm = layers.layer_norm_backward(first.x, saved.x, saved.norm.mean, saved.norm.rstd,
                                          self.norm_weight, residual_gradient=dy)
        return norm.x, [norm.weight, norm.bias, first.weight, first.bias, second.weight, second.bias]


class UpdateNetwork:
    """`blocks` UpdateBlocks over perception features and a normalised readout
    that is added to the particles' states."""

    def __init__(self, features: int, hidden: int, state_dims: int, blocks: int = 2,
                 activation: Activation = Activation.Gelu, dtype=None, device=None, seed: int = 0):
        import torch

        if blocks < 0 or state_dims < 1:
            raise InvalidArgument("blocks must be >= 0 and state_dims >= 1")
        dtype = dtype or torch.bfloat16
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        generator = torch.Generator(device=device)
        generator.manual_seed(seed)
        self.blocks = [UpdateBlock(features, hidden, activation, dtype, device, generator)
                       for _ in range(blocks)]
        self.eps = 1e-5
        self.norm_weight = torch.ones(features, dtype=dtype, device=device)
        self.norm_bias = torch.zeros(features, dtype=dtype, device=device)
        self.readout = _randn((state_dims, features), 0.1 * (1.0 / features) ** 0.5, dtype, device,
                              generator)
        self.readout_bias = torch.zeros(state_dims, dtype=dtype, device=device)

    def parameters(self) -> List["torch.Tensor"]:
        return [p for b in self.blocks for p in b.parameters()] + [
            self.norm_weight, self.norm_bias, self.readout, self.readout_bias]

    def forward(self, features, states, save: bool = True):
        """(next states, what backward reads or None)."""
        h, saved = features, []
        for block in self.blocks:
            h, s = block.forward(h, save)
            saved.append(s)
        norm = layers.layer_norm(h, self.norm_weight, self.norm_bias, self.eps)
        out = layers.linear(norm.y, self.readout, self.readout_bias, residual=states).y
        return out, ((saved, h, norm) if save else None)

    def backward(self, dy, saved):
        """(gradient of the features, gradient of the states, gradients in
        parameters()'s order)."""
        block_saved, h, norm = saved
        g = layers.linear_backward(dy, norm.y, self.readout)
        n = layers.layer_norm_backward(g.x, h, norm.mean, norm.rstd, self.norm_weight)
        dh, grads = n.x, [n.weight, n.bias, g.weight, g.bias]
        for block, s in zip(reversed(self.blocks), reversed(block_saved)):
            dh, block_grads = block.backward(dh, s)
            grads = block_grads + grads
        return dh, dy, grads

    def sgd_step(self, gradients, learning_rate: float) -> None:
        for p, g in zip(self.parameters(), gradients):
            p.sub_(g, alpha=float(learning_rate))
