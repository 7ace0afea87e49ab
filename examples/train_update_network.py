"""Trains a wide update network on what an NPA model does to its particles.

    python examples/train_update_network.py [--particles 4096] [--steps 60] [--dtype bf16]

The teacher is the 64 -> 128 -> 18 relu pair of the 2D growing configuration;
its perception features come from the library's hashgrid and perception
kernels, its raw update from npa_dev_model_forward_update.  The student is an
UpdateNetwork (layer norm, linear layers with activation and residual, and
their backward passes) fitted to next state = state + update by plain SGD.
"""

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import numpy as np  # noqa: E402
import torch  # noqa: E402

import burn_automata_b200 as ba  # noqa: E402
from burn_automata_b200 import _lib, workloads  # noqa: E402

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def teacher_data(particles: int, seed: int, device):
    """(features [n, F], states [n, C], next states [n, C]) in float32."""
    w = workloads.make("cfg0", seed, n=particles, steps=1)
    model = ba.NpaModel(w.model, ba.NpaWeights(w.weights.w1, w.weights.b1, w.weights.w2,
                                               w.weights.b2), device=device.index or 0)
    positions = torch.from_numpy(np.ascontiguousarray(w.positions)).to(device)
    states = torch.from_numpy(np.ascontiguousarray(w.states)).to(device)
    perceive = ba.DevicePerception(w.grid, w.model.perception_options(), 1, w.n,
                                   w.model.state_dims, device=device.index or 0)
    features, _ = perceive(positions, states)
    update = torch.empty(w.n * w.model.update_dims(), dtype=torch.float32, device=device)
    _lib.check(_lib.lib().npa_dev_model_forward_update(
        model.handle, features.data_ptr(), w.n, update.data_ptr(),
        torch.cuda.current_stream(device).cuda_stream), "forward_update")
    update = update.view(w.n, -1)[:, w.model.spatial_dims:]
    states = states.view(w.n, -1)
    torch.cuda.synchronize(device)
    model.close()
    return features.view(w.n, -1).clone(), states, states + update


def train(particles: int = 4096, steps: int = 60, dtype=torch.bfloat16, hidden: int = 512,
          blocks: int = 2, learning_rate: float = 0.01, seed: int = 0, log=print):
    """The mean squared error before each step."""
    device = torch.device("cuda", torch.cuda.current_device())
    features, states, target = (t.to(dtype) for t in teacher_data(particles, seed, device))
    net = ba.UpdateNetwork(features.shape[1], hidden, states.shape[1], blocks, dtype=dtype,
                           device=device, seed=seed)
    losses = []
    for step in range(steps):
        out, saved = net.forward(features, states)
        error = out.float() - target.float()
        losses.append(float(error.square().mean()))
        # the gradient of the summed squares per particle, averaged over particles
        dy = (error * (2.0 / particles)).to(dtype)
        _, _, gradients = net.backward(dy, saved)
        ba.check_layer_waits()  # a step whose kernels gave up must not reach the weights
        net.sgd_step(gradients, learning_rate)
        if log and (step % 10 == 0 or step + 1 == steps):
            log(f"step {step:4d}  mean squared error {losses[-1]:.5f}")
    return losses


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--particles", type=int, default=4096)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    p.add_argument("--hidden", type=int, default=512)
    p.add_argument("--blocks", type=int, default=2)
    a = p.parse_args()
    train(a.particles, a.steps, DTYPES[a.dtype], a.hidden, a.blocks)
