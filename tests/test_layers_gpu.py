"""Layer norm and the linear layer against plain 64-bit forms.

Tolerances.  u is the storage type's unit roundoff (2^-24, 2^-11, 2^-8): one
rounding of the result costs u |ref|.  A sum of K products held in f32 in
any order errs by about sqrt(K) roundings of its running value; it is granted
(sqrt(K) + 16) 2^-22 times the sum of the terms' magnitudes (the tensor cores
truncate where the f32 units round, hence 2^-22 and not 2^-24).  linear's
backward pass in 16 bits also rounds dz once, u times the magnitudes.
Activations and their slopes are granted 2^-20 (|z| + 1) per unit.
"""

import numpy as np
import pytest

import burn_automata_b200 as ba
from burn_automata_b200 import Activation

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# below the smallest normal number one rounding costs an absolute amount
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
EPS = 1e-5


def make(shape, dtype, seed, scale=1.0, shift=0.0, pitch=0, offset=0):
    """Seeded normal values; pitch widens the rows' buffer, offset moves its start."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    width = shape[-1] + pitch
    rows = int(np.prod(shape[:-1], dtype=np.int64)) if len(shape) > 1 else 1
    flat = torch.empty(rows * width + offset, device="cuda").normal_(shift, scale, generator=gen)
    t = flat.to(dtype)[offset:].view(*shape[:-1], width) if len(shape) > 1 else \
        flat.to(dtype)[offset:offset + shape[0]]
    return t[..., :shape[-1]]


def close(got, ref, bound, name):
    got = got.double()
    assert got.shape == ref.shape, name
    limit = bound + UNIT_OF * ref.abs() + TINY_OF
    bad = ~((got - ref).abs() <= limit)
    if bool(bad.any()):
        i = int(((got - ref).abs() - limit).nan_to_num(float("inf")).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {ref.numel()} outside, worst at {i}: "
                             f"{got.reshape(-1)[i].item()} for {ref.reshape(-1)[i].item()}, "
                             f"allowed {limit.reshape(-1)[i].item()}")


def set_type(dtype):
    global UNIT_OF, TINY_OF
    UNIT_OF, TINY_OF = UNIT[dtype], TINY[dtype]


def sum_error(k):
    return (k ** 0.5 + 16) * 2.0 ** -22


# ------------------------------------------------------------------ layer norm
NORMS = [  # rows, dims, pitch, offset
    (1, 1, 0, 0), (1, 7, 0, 0), (5, 8, 0, 0), (33, 16, 0, 0), (4096, 64, 0, 0), (257, 64, 1, 0),
    (100, 130, 0, 0), (1000, 130, 0, 1), (64, 160, 0, 0), (65, 160, 8, 3), (17, 512, 0, 0),
    (9, 513, 0, 0), (300, 1024, 0, 0), (7, 1025, 3, 1), (40, 4096, 0, 0), (5, 4095, 0, 0),
    (3, 8192, 24, 0), (4, 8191, 0, 0), (2, 20000, 0, 0), (3, 16385, 1, 1), (20000, 36, 0, 0),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,dims,pitch,offset", NORMS)
def test_layer_norm(rows, dims, pitch, offset, dtype):
    dt = TYPES[dtype]
    set_type(dt)
    x = make((rows, dims), dt, 1, 2.0, 0.5, pitch, offset)
    w = make((dims,), dt, 2, 0.2, 1.0) if dims % 3 else None
    b = make((dims,), dt, 3, 0.2) if dims % 5 else None
    out = ba.layer_norm(x, w, b, EPS)
    xd = x.double()
    mean = xd.mean(1, keepdim=True)
    rstd = 1 / ((xd - mean).pow(2).mean(1, keepdim=True) + EPS).sqrt()
    wd = w.double() if w is not None else torch.ones(dims, device="cuda").double()
    bd = b.double() if b is not None else torch.zeros(dims, device="cuda").double()
    ref = (xd - mean) * rstd * wd + bd
    size = xd.abs().amax(1, keepdim=True) * rstd
    e = sum_error(dims)
    close(out.y, ref, e * (wd.abs() * size + bd.abs()), "y")
    set_type(torch.float32)
    close(out.mean, mean[:, 0], e * xd.abs().mean(1), "mean")
    close(out.rstd, rstd[:, 0], e * rstd[:, 0] * (1 + size[:, 0]), "rstd")


@pytest.mark.parametrize("dims", [62, 64, 128, 130, 144, 146])
def test_layer_norm_rings_of_every_depth(dims):
    """f32 widths on both sides of the forward ring's choices of tile and depth;
    enough rows that a ring turns, and a last tile that is not whole."""
    test_layer_norm(75779, dims, 0, 0, next(k for k, v in TYPES.items() if v == torch.float32))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,dims,pitch,offset", NORMS)
def test_layer_norm_backward(rows, dims, pitch, offset, dtype):
    dt = TYPES[dtype]
    x = make((rows, dims), dt, 1, 2.0, 0.5, pitch, offset)
    dy = make((rows, dims), dt, 4, 1.0, 0.1, 0, offset)
    w = make((dims,), dt, 2, 0.2, 1.0) if dims % 3 else None
    res = make((rows, dims), dt, 5, 1.0, 0.0, pitch) if rows % 2 else None
    saved = ba.layer_norm(x, w, None, EPS)
    g = ba.layer_norm_backward(dy, x, saved.mean, saved.rstd, w, residual_gradient=res,
                               needs=("x", "weight", "bias"))
    set_type(dt)
    m, r = saved.mean.double()[:, None], saved.rstd.double()[:, None]
    xh = (x.double() - m) * r
    dyd = dy.double()
    wd = w.double() if w is not None else torch.ones(dims, device="cuda").double()
    gg = dyd * wd
    ref = r * (gg - gg.mean(1, keepdim=True) - xh * (gg * xh).mean(1, keepdim=True))
    size = (x.double().abs() + m.abs()) * r  # what xhat's cancellation leaves
    terms = r * (gg.abs() + gg.abs().mean(1, keepdim=True)
                 + (1 + size) * (gg.abs() * (1 + size)).mean(1, keepdim=True))
    if res is not None:
        ref = ref + res.double()
        terms = terms + res.double().abs()
    close(g.x, ref, sum_error(dims) * terms, "dx")
    close(g.weight, (dyd * xh).sum(0), sum_error(rows) * (dyd.abs() * (xh.abs() + size)).sum(0),
          "dweight")
    close(g.bias, dyd.sum(0), sum_error(rows) * dyd.abs().sum(0), "dbias")


def test_layer_norm_gradient_against_differences():
    """d/dh of sum(c y(x + h v)) against <dx, v>: the central difference errs by
    h^2 / 6 times the third derivative (order one here) and 2^-24 sqrt(n) / h
    of rounding, both below 2e-4 at h = 2^-6."""
    x, c = make((7, 96), torch.float32, 1), make((7, 96), torch.float32, 2)
    w, b = make((96,), torch.float32, 3, 0.2, 1.0), make((96,), torch.float32, 4)
    o = ba.layer_norm(x, w, b)
    g = ba.layer_norm_backward(c, x, o.mean, o.rstd, w)
    h = 2.0 ** -6

    def slope(f, v):
        up, down = f(h * v), f(-h * v)
        return float(((up - down).double() * c.double()).sum() / (2 * h))

    for seed, got, f, shape in (
            (5, g.x, lambda d: ba.layer_norm(x + d, w, b).y, x.shape),
            (6, g.weight, lambda d: ba.layer_norm(x, w + d, b).y, w.shape),
            (7, g.bias, lambda d: ba.layer_norm(x, w, b + d).y, b.shape)):
        v = make(tuple(shape), torch.float32, seed)
        want = slope(f, v)
        have = float((got.double() * v.double()).sum())
        assert abs(have - want) <= 1e-3 * float(got.double().norm() * v.double().norm())


def test_layer_norm_keeps_the_spread_of_rows_far_from_zero():
    x = make((64, 256), torch.float32, 1, 1e-2, 1000.0)
    xd = x.double()
    ref = 1 / (xd.var(1, correction=0) + EPS).sqrt()
    got = ba.layer_norm(x).rstd.double()
    # the values themselves are multiples of 2^-14; the mean rounds to 2^-15
    assert float(((got - ref) / ref).abs().max()) <= 1e-4


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dims", [64, 130, 4096])
def test_layer_norm_rows_with_nan_or_infinity_stay_alone(dtype, dims):
    x = make((20, dims), TYPES[dtype], 1)
    clean = ba.layer_norm(x).y
    x[3, 5] = float("nan")
    x[11, dims - 1] = float("inf")
    y = ba.layer_norm(x).y
    for r in range(20):
        if r in (3, 11):
            assert bool(y[r].isnan().all())
        else:
            assert torch.equal(y[r], clean[r])


# ---------------------------------------------------------------------- linear
LINEARS = [  # rows, inputs, outputs, pitch, offset
    (1, 1, 1, 0, 0), (1, 64, 128, 0, 0), (2, 7, 3, 0, 0), (3, 1024, 512, 0, 0),
    (8, 4096, 72, 0, 0), (9, 333, 65, 1, 1), (31, 160, 256, 0, 0), (127, 64, 64, 0, 0),
    (128, 64, 128, 0, 0), (129, 72, 136, 8, 0), (1000, 160, 256, 0, 0), (1000, 256, 35, 0, 0),
    (515, 130, 18, 0, 0), (515, 128, 18, 8, 3), (4096, 64, 128, 0, 0), (300, 1000, 264, 24, 0),
    (640, 512, 1024, 0, 0), (257, 2048, 255, 0, 0), (20000, 16, 8, 0, 0), (33000, 64, 128, 0, 0),
    (20001, 24, 40, 0, 0), (130, 8, 2000, 0, 0), (64, 33, 513, 7, 5),
]


def act64(z, act):
    if act == Activation.Relu:
        return z.clamp(min=0), (z > 0).double()
    if act == Activation.Gelu:
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if act == Activation.GeluTanh:
        k = np.sqrt(2 / np.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k
                                   * (1 + 3 * 0.044715 * z * z))
    if act == Activation.Silu:
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,inputs,outputs,pitch,offset", LINEARS)
def test_linear(rows, inputs, outputs, pitch, offset, dtype):
    dt = TYPES[dtype]
    set_type(dt)
    act = Activation((rows + outputs) % 5)
    x = make((rows, inputs), dt, 1, 1.0, 0.1, pitch, offset)
    w = make((outputs, inputs), dt, 2, (2.0 / inputs) ** 0.5, 0.0, pitch, offset)
    b = make((outputs,), dt, 3, 0.5) if outputs % 3 else None
    res = make((rows, outputs), dt, 4, 1.0, 0.0, pitch) if rows % 2 else None
    out = ba.linear(x, w, b, residual=res, activation=act, save_pre_activation=inputs % 2 == 0)
    z = x.double() @ w.double().t()
    size = sum_error(inputs) * (x.double().abs() @ w.double().abs().t())
    if b is not None:
        z = z + b.double()
        size = size + 2.0 ** -23 * b.double().abs()
    y = act64(z, act)[0]
    if res is not None:
        y = y + res.double()
        size_y = size + 2.0 ** -23 * res.double().abs()
    else:
        size_y = size
    close(out.y, y, 1.2 * size_y + 2.0 ** -20 * (z.abs() + 1), "y")
    if inputs % 2 == 0:
        close(out.pre_activation, z, size, "z")
    else:
        assert out.pre_activation is None


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,inputs,outputs,pitch,offset", LINEARS)
def test_linear_backward(rows, inputs, outputs, pitch, offset, dtype):
    dt = TYPES[dtype]
    set_type(dt)
    act = Activation((rows + inputs) % 5)
    x = make((rows, inputs), dt, 1, 1.0, 0.1, pitch, offset)
    w = make((outputs, inputs), dt, 2, (2.0 / inputs) ** 0.5, 0.0, pitch, offset)
    dy = make((rows, outputs), dt, 3, 1.0, 0.1, pitch, offset)
    z = make((rows, outputs), dt, 4, 1.4, 0.0, 0, offset)
    g = ba.linear_backward(dy, x, w, z if act else None, activation=act)
    slope = act64(z.double(), act)[1]
    dz = dy.double() * slope
    # dz is rounded to 16 bits for the products; the slope errs by 2^-20 (|z| + 1)
    rounded = 0.0 if act == Activation.Identity or dt == torch.float32 else UNIT[dt]
    dz_err = (dz.abs() * rounded + (dy.double().abs() * 2.0 ** -20 * (z.double().abs() + 1)
                                    if act else 0.0))
    wa, xa = w.double().abs(), x.double().abs()
    close(g.x, dz @ w.double(), sum_error(outputs) * (dz.abs() @ wa) + dz_err @ wa
          if act else sum_error(outputs) * (dz.abs() @ wa), "dx")
    close(g.weight, dz.t() @ x.double(), sum_error(rows) * (dz.abs().t() @ xa) + dz_err.t() @ xa
          if act else sum_error(rows) * (dz.abs().t() @ xa), "dweight")
    close(g.bias, dz.sum(0), sum_error(rows) * dz.abs().sum(0)
          + (dz_err.sum(0) if act else 0.0), "dbias")


@pytest.mark.parametrize("act", list(Activation))
def test_linear_gradient_against_differences(act):
    """As for layer norm; relu's kink costs h per crossing value, so its
    directional difference is granted ten times more."""
    x, w = make((9, 40), torch.float32, 1), make((24, 40), torch.float32, 2, 0.2)
    b, c = make((24,), torch.float32, 3), make((9, 24), torch.float32, 4)
    o = ba.linear(x, w, b, activation=act, save_pre_activation=True)
    g = ba.linear_backward(c, x, w, o.pre_activation, activation=act)
    h = 2.0 ** -6
    for seed, got, f in (
            (5, g.x, lambda d: ba.linear(x + d, w, b, activation=act).y),
            (6, g.weight, lambda d: ba.linear(x, w + d, b, activation=act).y),
            (7, g.bias, lambda d: ba.linear(x, w, b + d, activation=act).y)):
        v = make(tuple(got.shape), torch.float32, seed)
        v = v / v.norm() * got.numel() ** 0.25
        want = float(((f(h * v) - f(-h * v)).double() * c.double()).sum() / (2 * h))
        have = float((got.double() * v.double()).sum())
        limit = 1e-2 if act == Activation.Relu else 1e-3
        assert abs(have - want) <= limit * float(got.double().norm() * v.double().norm())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [4, 200])
def test_linear_infinities_and_nan(dtype, rows):
    """Infinite and NaN inputs reach the outputs that they belong to, as in
    64-bit arithmetic, and no other."""
    dt = TYPES[dtype]
    x, w = make((rows, 96), dt, 1), make((40, 96), dt, 2, 0.2)
    w = torch.where(w == 0, torch.ones_like(w), w)
    x[1, 3], x[2, 95] = float("inf"), float("nan")
    w[7, 10] = float("-inf")
    got = ba.linear(x, w).y.double()
    ref = x.double() @ w.double().t()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.isinf() & (got > 0), ref.isinf() & (ref > 0))
    assert torch.equal(got.isinf() & (got < 0), ref.isinf() & (ref < 0))
    g = ba.linear_backward(make((rows, 40), dt, 3), x, w)
    dyd = make((rows, 40), dt, 3).double()
    for have, want in ((g.x.double(), dyd @ w.double()), (g.weight.double(), dyd.t() @ x.double())):
        assert torch.equal(have.isnan(), want.isnan())
        assert torch.equal(have.isinf(), want.isinf())


def test_linear_large_and_small_values_in_f32():
    """Products near the ends of the f32 range keep f32's relative accuracy."""
    for sx, sw in ((1e30, 1e-25), (1e-25, 1e20), (3e38, 1e-3), (1e-20, 1e-12)):
        x, w = make((150, 64), torch.float32, 1), make((40, 64), torch.float32, 2)
        x, w = (x / x.abs().max() * sx), (w / w.abs().max() * sw)
        ref = x.double() @ w.double().t()
        size = x.double().abs() @ w.double().abs().t()
        err = ((ba.linear(x, w).y.double() - ref).abs() / size).max()
        assert float(err) <= sum_error(64), (sx, sw)


# ------------------------------------------------------------- ways of calling
def test_no_rows():
    x = torch.zeros((0, 24), device="cuda")
    w = torch.ones((8, 24), device="cuda")
    o = ba.layer_norm(x, torch.ones(24, device="cuda"))
    assert o.y.shape == (0, 24) and o.mean.shape == (0,)
    g = ba.layer_norm_backward(x, x, o.mean, o.rstd, torch.ones(24, device="cuda"))
    assert g.x.shape == (0, 24)
    assert float(g.weight.abs().sum()) == 0.0 and float(g.bias.abs().sum()) == 0.0
    assert ba.linear(x, w).y.shape == (0, 8)
    dy = torch.zeros((0, 8), device="cuda")
    g = ba.linear_backward(dy, x, w, dy, activation=Activation.Gelu)
    assert g.x.shape == (0, 24)
    assert float(g.weight.abs().sum()) == 0.0 and float(g.bias.abs().sum()) == 0.0


def test_leading_axes_and_other_orders():
    x = make((6, 5, 48), torch.float32, 1)
    w = make((32, 48), torch.float32, 2, 0.2)
    y = ba.linear(x, w).y
    assert y.shape == (6, 5, 32)
    flat = ba.linear(x.reshape(30, 48), w).y
    assert torch.equal(y.reshape(30, 32), flat)
    assert torch.equal(ba.linear(x.transpose(0, 1), w).y, y.transpose(0, 1))
    assert torch.equal(ba.linear(x, w.t().contiguous().t()).y, y)
    o = ba.layer_norm(x.transpose(0, 1))
    assert torch.equal(o.y, ba.layer_norm(x).y.transpose(0, 1)) and o.mean.shape == (5, 6)
    one = ba.linear(x[0, 0], w).y
    assert one.shape == (32,)
    row = x[:1, 0].expand(7, 48)  # stride 0
    assert torch.equal(ba.layer_norm(row).y[6], ba.layer_norm(x[:1, 0]).y[0])


@pytest.mark.parametrize("needs", [("x",), ("weight",), ("bias",), ("x", "bias"), ()])
def test_only_the_needed_gradients(needs):
    x, dy = make((70, 48), torch.bfloat16, 1), make((70, 24), torch.bfloat16, 2)
    w, z = make((24, 48), torch.bfloat16, 3), make((70, 24), torch.bfloat16, 4)
    full = ba.linear_backward(dy, x, w, z, activation=Activation.Silu)
    part = ba.linear_backward(dy, x, w, z, activation=Activation.Silu, needs=needs)
    for k in ("x", "weight", "bias"):
        a, b = getattr(full, k), getattr(part, k)
        assert (b is None) == (k not in needs)
        assert b is None or torch.equal(a, b)
    o = ba.layer_norm(x)
    ones = torch.ones(48, device="cuda", dtype=torch.bfloat16)
    full = ba.layer_norm_backward(x, x, o.mean, o.rstd, ones)
    part = ba.layer_norm_backward(x, x, o.mean, o.rstd, ones, needs=needs)
    for k in ("x", "weight", "bias"):
        a, b = getattr(full, k), getattr(part, k)
        assert (b is None) == (k not in needs)
        assert b is None or torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows 65,536 values apart: the last ones lie past 2^31 elements."""
    rows, pitch = 33500, 1 << 16
    big = torch.empty(rows * pitch, dtype=torch.float16, device="cuda")
    x = big.view(rows, pitch)[:, 128:128 + 64]
    x.copy_(make((rows, 64), torch.float16, 1))
    w = make((32, 64), torch.float16, 2, 0.2)
    dense = x.contiguous()
    assert torch.equal(ba.layer_norm(x).y, ba.layer_norm(dense).y)
    assert torch.equal(ba.linear(x, w).y, ba.linear(dense, w).y)
    dy = make((rows, 32), torch.float16, 3)
    a, b = ba.linear_backward(dy, x, w), ba.linear_backward(dy, dense, w)
    assert torch.equal(a.weight, b.weight) and torch.equal(a.x, b.x)


def all_calls(x, w, dy, z):
    o = ba.layer_norm(x, x[0].contiguous())
    g = ba.layer_norm_backward(x, x, o.mean, o.rstd, x[0].contiguous())
    y = ba.linear(x, w, activation=Activation.Gelu, save_pre_activation=True)
    d = ba.linear_backward(dy, x, w, z, activation=Activation.Gelu)
    return [o.y, o.mean, o.rstd, g.x, g.weight, g.bias, y.y, y.pre_activation, d.x, d.weight,
            d.bias]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_same_results_again_on_another_stream_and_in_a_graph(dtype):
    dt = TYPES[dtype]
    x, w = make((3000, 160), dt, 1), make((96, 160), dt, 2, 0.1)
    dy, z = make((3000, 96), dt, 3), make((3000, 96), dt, 4)
    first = all_calls(x, w, dy, z)
    for a, b in zip(first, all_calls(x, w, dy, z)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = all_calls(x, w, dy, z)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = all_calls(x, w, dy, z)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, captured):
        assert torch.equal(a, b)


def test_shapes_types_and_devices_that_do_not_fit():
    x, w = make((4, 16), torch.float32, 1), make((8, 16), torch.float32, 2)
    bad = [
        lambda: ba.linear(x, w[:, :8]), lambda: ba.linear(x, w.half()),
        lambda: ba.linear(x, w.cpu()), lambda: ba.linear(x, w, w[0]),
        lambda: ba.linear(x, w, residual=x), lambda: ba.linear(x.double(), w),
        lambda: ba.linear(x, w, activation=9), lambda: ba.linear(x, w[0]),
        lambda: ba.linear_backward(x, x, w),
        lambda: ba.linear_backward(ba.linear(x, w).y, x, w, activation=Activation.Relu),
        lambda: ba.linear_backward(ba.linear(x, w).y, x, w, needs=("y",)),
        lambda: ba.layer_norm(x, w), lambda: ba.layer_norm(x, w[0].half()),
        lambda: ba.layer_norm_backward(x, x, x[:, 0].half(), x[:, 0].contiguous()),
        lambda: ba.layer_norm_backward(x, x, x[:3, 0].contiguous(), x[:, 0].contiguous()),
        lambda: ba.layer_norm_backward(x, x, x[:, 0].contiguous(), x[:, 0].contiguous(),
                                       residual_gradient=x, needs=("bias",)),
    ]
    for call in bad:
        with pytest.raises(ba.KernelError):
            call()
    with pytest.raises(ba.config.InvalidEps):
        ba.layer_norm(x, eps=0.0)


# Shapes at which the linear layer changes its way of working: odd widths with
# enough work to be packed, tiles of block pairs with ragged edges, small layers
# over many rows (the one-walk backward pass), every count of few rows.
WAYS = [  # rows, inputs, outputs
    (9000, 251, 240), (4200, 513, 384), (2100, 515, 1000), (2049, 1024, 1030), (300, 264, 4104),
    (257, 4096, 520), (2048, 64, 192), (5001, 160, 64), (2500, 256, 64), (3333, 96, 256),
    (6000, 200, 16), (10000, 8, 8), (4444, 72, 120),
] + [(r, 1000, 2100) for r in range(1, 10)] + [(r, 77, 50) for r in (3, 5, 8)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,inputs,outputs", WAYS)
def test_linear_at_its_ways_borders(rows, inputs, outputs, dtype):
    test_linear(rows, inputs, outputs, 0, 0, dtype)
    test_linear_backward(rows, inputs, outputs, 0, 0, dtype)


def test_waits_all_end():
    """No bounded wait of the kernels above has given up."""
    assert ba.load_library().npa_bulk_copy_timeouts() == 0
