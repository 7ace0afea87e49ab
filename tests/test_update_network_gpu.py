"""The update network: its passes against 64-bit autograd, and training it on
what an NPA model does to its particles."""

import sys
from pathlib import Path

import pytest

import burn_automata_b200 as ba

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACTS = {ba.Activation.Identity: lambda z: z, ba.Activation.Relu: torch.relu,
        ba.Activation.Gelu: torch.nn.functional.gelu,
        ba.Activation.GeluTanh: lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
        ba.Activation.Silu: torch.nn.functional.silu}


def activate(act, z, saved_z):
    """act(z) whose slope is taken at the pre-activation that the network kept, as
    its backward pass does: relu's slope jumps where rounding moves z across zero."""
    at = saved_z.detach().double().requires_grad_()
    slope, = torch.autograd.grad(ACTS[act](at).sum(), at)
    return ACTS[act](z).detach() + slope * (z - z.detach())


def reference(net, features, states, saved):
    """The same network in float64 with autograd: (output, leaves)."""
    leaves = [t.detach().double().requires_grad_() for t in [features, states] + net.parameters()]
    h, it = leaves[0], iter(leaves[2:])
    norm = torch.nn.functional.layer_norm
    for block, kept in zip(net.blocks, saved[0]):
        nw, nb, w1, b1, w2, b2 = (next(it) for _ in range(6))
        z = norm(h, h.shape[-1:], nw, nb, block.eps) @ w1.t() + b1
        h = h + activate(block.activation, z, kept.hidden.pre_activation) @ w2.t() + b2
    nw, nb, w, b = (next(it) for _ in range(4))
    return leaves[1] + norm(h, h.shape[-1:], nw, nb, net.eps) @ w.t() + b, leaves


@pytest.mark.parametrize("dtype,tolerance", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2),
                                             (torch.float16, 4e-3)], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,features,hidden,state,act", [
    (4096, 64, 128, 16, ba.Activation.Relu), (1000, 130, 512, 32, ba.Activation.Gelu),
    (1, 64, 96, 16, ba.Activation.Silu), (2500, 160, 256, 35, ba.Activation.GeluTanh)])
def test_passes_match_autograd(rows, features, hidden, state, act, dtype, tolerance):
    """Normwise: some ten roundings to the storage type lie on the path, each
    2^-24, 2^-8 or 2^-11 of what it rounds."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    net = ba.UpdateNetwork(features, hidden, state, 2, act, dtype, seed=1)
    for p in net.parameters():
        p.add_(torch.randn(p.shape, generator=gen, device="cuda").to(dtype) * 0.02)
    x = torch.randn(rows, features, generator=gen, device="cuda").to(dtype)
    s = torch.randn(rows, state, generator=gen, device="cuda").to(dtype)
    dy = torch.randn(rows, state, generator=gen, device="cuda").to(dtype)
    out, saved = net.forward(x, s)
    dx, ds, grads = net.backward(dy, saved)
    ref, leaves = reference(net, x, s, saved)
    ref.backward(dy.double())
    got = [out, dx, ds] + grads
    want = [ref.detach()] + [t.grad for t in leaves]
    assert len(got) == len(want)
    for i, (g, r) in enumerate(zip(got, want)):
        assert g.shape == r.shape
        assert float((g.double() - r).norm() / r.norm()) <= tolerance, i
    again, none = net.forward(x, s, save=False)
    assert none is None and torch.equal(again, out)


def test_training_follows_the_model():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import train_update_network

    for dtype in (torch.float32, torch.bfloat16):
        losses = train_update_network.train(2048, 40, dtype, hidden=256, log=None)
        assert losses[-1] < 0.5 * losses[0]
        assert all(b < 1.5 * a for a, b in zip(losses, losses[1:]))


def test_refusals():
    with pytest.raises(ba.KernelError):
        ba.UpdateNetwork(0, 8, 4)
    with pytest.raises(ba.KernelError):
        ba.UpdateNetwork(8, 8, 4, blocks=-1)
    net = ba.UpdateNetwork(8, 16, 4)
    with pytest.raises(ba.KernelError):
        net.forward(torch.zeros(3, 9, dtype=torch.bfloat16, device="cuda"),
                    torch.zeros(3, 4, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ba.KernelError):
        net.forward(torch.zeros(3, 8, device="cuda"), torch.zeros(3, 4, device="cuda"))
