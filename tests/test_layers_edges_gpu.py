"""Layer norm and the linear layer where values, lengths and addresses are out
of the ordinary: infinities and NaN over long sums, sums of many thousand terms
of one sign, activations far out on their tails, views that start anywhere.

The tolerances are those of test_layers_gpu.py unless a test derives its own.
"""

import pytest

import burn_automata_b200 as ba
from burn_automata_b200 import Activation

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def normal(shape, dtype, seed, scale=1.0, shift=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(shift, scale, generator=gen).to(dtype)


def uniform(shape, dtype, seed, low, high):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.empty(shape, device="cuda").uniform_(low, high, generator=gen).to(dtype)


def waits_that_gave_up():
    torch.cuda.synchronize()
    return ba.load_library().npa_bulk_copy_timeouts()


# ------------------------------------------------- infinities and NaN in f32
def test_f32_weight_gradient_of_a_diverged_step():
    """Every gradient NaN, or infinite, over a long sum: the same walk as for
    finite values, with no wait that gives up."""
    rows, inputs, outputs = 300000, 640, 520
    x, w = normal((rows, inputs), F32, 1), normal((outputs, inputs), F32, 2, 0.05)
    before = waits_that_gave_up()
    for value in (NAN, INF, -INF):
        dy = torch.full((rows, outputs), value, device="cuda")
        g = ba.linear_backward(dy, x, w)
        # x and w have both signs: infinities of both signs meet in every sum
        assert bool(g.weight.isnan().all()) and bool(g.x.isnan().all())
        assert bool(g.bias.isnan().all()) if value != value else bool((g.bias == value).all())
    assert waits_that_gave_up() == before


def test_f32_infinities_at_the_end_of_a_long_sum():
    rows, inputs, outputs = 200003, 96, 72
    x, w = normal((rows, inputs), F32, 1), normal((outputs, inputs), F32, 2, 0.1)
    dy = normal((rows, outputs), F32, 3)
    dy = torch.where(dy == 0, torch.ones_like(dy), dy)
    clean = ba.linear_backward(dy, x, w).weight
    x[-1, 3] = INF                      # one infinite term: its sign
    x[-2, 7], x[5, 7] = INF, NAN        # a NaN wins
    x[1000, 11], x[-7, 11] = INF, -INF  # sign by the gradients' signs, NaN where they meet
    dy[-1, 9] = 0.0                     # an infinity times zero
    got = ba.linear_backward(dy, x, w).weight
    assert torch.equal(got[:9, 3], dy[-1, :9] * INF) and torch.equal(got[10:, 3], dy[-1, 10:] * INF)
    assert bool(got[9, 3].isnan())
    assert bool(got[:, 7].isnan().all())
    want = dy[1000] * INF + dy[-7] * -INF
    assert torch.equal(got[:, 11].isnan(), want.isnan())
    assert torch.equal(got[:, 11].nan_to_num(0.0, INF, -INF), want.nan_to_num(0.0, INF, -INF))
    other = [c for c in range(inputs) if c not in (3, 7, 11)]
    keep = [r for r in range(outputs) if r != 9]
    assert torch.equal(got[keep][:, other], clean[keep][:, other])


@pytest.mark.parametrize("rows", [200, 3000])
@pytest.mark.parametrize("inputs", [16, 97, 1000])
def test_f32_infinities_and_nan_where_64_bits_have_them(rows, inputs):
    """Against 64-bit products, entry by entry; a payload in a NaN's low bits
    alone, which a cut to 16 bits would lose, among them."""
    x, w = normal((rows, inputs), F32, 1), normal((40, inputs), F32, 2, 0.2)
    w[3] = 1.0  # whole in 16 bits: nothing is left for its second and third part
    w[5, 4], w[6, 4] = 0.0, INF
    x[1, 4], x[2, 4], x[4, inputs - 1] = INF, -INF, NAN
    x[7, 2], x[7, 9] = INF, -INF
    x.view(torch.int32)[9, 3] = 0x7F800001
    x.view(torch.int32)[10, 3] = 0x7F800001 - (1 << 31)
    got, ref = ba.linear(x, w).y.double(), x.double() @ w.double().t()
    ref[9:11] = NAN
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.isinf() & (got > 0), ref.isinf() & (ref > 0))
    assert torch.equal(got.isinf() & (got < 0), ref.isinf() & (ref < 0))


def test_f32_largest_values():
    """Values up to the largest f32 stay finite where their products are."""
    x, w = torch.zeros((150, 64), device="cuda"), torch.zeros((40, 64), device="cuda")
    top = torch.finfo(F32).max
    x[:, 5], w[:, 5] = top, 0.5
    x[3, 5], w[7, 5] = -top, -1.0
    ref = x.double() @ w.double().t()
    got = ba.linear(x, w).y.double()
    assert bool(((got - ref).abs() <= 2.0 ** -22 * ref.abs()).all())


# ------------------------------------------- long sums of terms of one sign
def one_sign_error(k):
    """What a 16-bit product's sum of k terms of one sign may lose, relative to
    their sum: 512 accumulating steps of the tensor core with a unit of 2^-23
    each, and the f32 sum of the parts."""
    return 2.0 ** -14 + (k / 4096) ** 0.5 * 2.0 ** -24


LONG = [  # rows, inputs, outputs: products whose k (the rows) is split or not
    (131149, 2048, 1280),  # pairs' tiles, k in one piece
    (262144, 1024, 512),   # pairs' tiles, split k
    (1000003, 9, 7),       # odd widths: loader warps
    (700001, 264, 24),     # one narrow tile, split k
    (70000, 1000, 2056),   # ragged tiles
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows,inputs,outputs", LONG)
def test_weight_gradient_of_many_rows_of_one_sign(rows, inputs, outputs, dtype):
    top = (40000.0 / rows) ** 0.5  # the sums stay inside f16
    x = uniform((rows, inputs), dtype, 1, top / 2, top)
    dy = uniform((rows, outputs), dtype, 2, top / 2, top)
    w = torch.zeros((outputs, inputs), dtype=dtype, device="cuda")
    got = ba.linear_backward(dy, x, w, needs=("weight",)).weight.double()
    ref = dy.double().t() @ x.double()
    unit = 2.0 ** -11 if dtype == F16 else 2.0 ** -8
    assert float(((got - ref).abs() / ref).max()) <= unit + one_sign_error(rows)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows,inputs,outputs", [(2048, 9000, 4096), (2100, 4160, 4099), (300, 40008, 136),
                                                 (1000, 4097, 40)])
def test_linear_of_many_inputs_of_one_sign(rows, inputs, outputs, dtype):
    """The same over many inputs, with the whole epilogue behind it."""
    top = (2000.0 / inputs) ** 0.5
    x, w = uniform((rows, inputs), dtype, 1, top / 2, top), uniform((outputs, inputs), dtype, 2, top / 2, top)
    b, res = uniform((outputs,), dtype, 3, 1, 2), uniform((rows, outputs), dtype, 4, 1, 2)
    out = ba.linear(x, w, b, residual=res, activation=Activation.Relu, save_pre_activation=True)
    z = x.double() @ w.double().t() + b.double()
    unit = 2.0 ** -11 if dtype == F16 else 2.0 ** -8
    for got, ref in ((out.pre_activation, z), (out.y, z + res.double())):
        assert float(((got.double() - ref).abs() / ref).max()) <= unit + one_sign_error(inputs)


def test_one_walk_backward_of_many_rows_of_one_sign():
    """Few weights and so many rows that a block's walk over them has to end
    more than once."""
    rows, inputs, outputs = 20000003, 16, 8
    top = (40000.0 / rows) ** 0.5
    x = uniform((rows, inputs), F16, 1, top / 2, top)
    dy = uniform((rows, outputs), F16, 2, top / 2, top)
    w = normal((outputs, inputs), F16, 3)
    g = ba.linear_backward(dy, x, w)
    ref = dy.double().t() @ x.double()
    assert float(((g.weight.double() - ref).abs() / ref).max()) <= 2.0 ** -11 + one_sign_error(rows)
    assert bool(g.bias.isinf().all())  # 670,000: beyond f16
    some = slice(0, rows, 99991)
    ref = dy[some].double() @ w.double()
    size = dy[some].double().abs() @ w.double().abs()
    assert bool(((g.x[some].double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -20 * size + 2.0 ** -24).all())


# ------------------------------------------------------------------- waits
def test_check_of_waits_after_healthy_calls():
    """Nothing gave up: the check waits for the stream and returns, however the
    device is named."""
    x, w = normal((300, 64), F16, 1), normal((32, 64), F16, 2)
    ba.linear(x, w)
    ba.check_layer_waits()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ba.layer_norm(x)
        ba.check_layer_waits("cuda:0")
        assert side.query()  # it waited
    ba.check_layer_waits(torch.device("cuda"))


def test_threads_with_new_shapes():
    """Threads whose first calls of a kernel come with different shapes, and so
    with different amounts of shared memory."""
    import threading

    widths = [64 + 4 * i for i in range(24)]
    x = {d: normal((5000, d), F32, d) for d in widths}
    w = normal((64, 64), BF16, 1)
    want = {d: torch.nn.functional.layer_norm(x[d].double(), (d,)) for d in widths}
    errors = []

    def work(part):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for d in part:
                    o = ba.layer_norm(x[d])
                    ba.layer_norm_backward(x[d], x[d], o.mean, o.rstd)
                    ba.linear(x[d][:, :64].bfloat16(), w)
                    assert float((o.y.double() - want[d]).abs().max()) < 1e-4
        except BaseException as e:  # noqa: BLE001 -- reported by the test's own thread
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(widths[i::6],)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors


# ------------------------------------------------------- activations' tails
def through_linear(z, act, rows):
    """act at the values z (one per output), through products of one-hot rows."""
    x, w = torch.zeros((rows, 16), dtype=z.dtype, device="cuda"), torch.zeros((z.numel(), 16), dtype=z.dtype,
                                                                              device="cuda")
    x[:, 0], w[:, 0] = 1, z
    return ba.linear(x, w, activation=act).y[rows - 1].double()


def slope_through_backward(z, act, rows):
    """act' at z as the bias gradient of one row of ones, and as an x gradient."""
    dy = torch.zeros((rows, z.numel()), dtype=z.dtype, device="cuda")
    dy[rows - 1] = 1
    x = torch.zeros((rows, 16), dtype=z.dtype, device="cuda")
    w = torch.zeros((z.numel(), 16), dtype=z.dtype, device="cuda")
    g = ba.linear_backward(dy, x, w, z.expand(rows, -1).contiguous(), activation=act, needs=("bias",))
    return g.bias.double()


def normal_cdf_and_density(z):
    # ndtr cancels below zero as 1 + erf does
    return torch.special.erfc(-z / 2 ** 0.5) / 2, torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5


@pytest.mark.parametrize("rows", [3, 200])
def test_f32_gelu_tail(rows):
    """z Phi(z) down to -12 with a relative error: the argument's two roundings
    move erfc by z^2 2^-23 of itself, the function and the products err by a few
    2^-23."""
    z = torch.linspace(-12, 8, 4001, device="cuda")
    cdf, density = normal_cdf_and_density(z.double())
    bound = 2.0 ** -20 + z.double() ** 2 * 2.0 ** -22
    got = through_linear(z, Activation.Gelu, rows)
    assert float(((got - z.double() * cdf).abs() / (z.double() * cdf).abs().clamp(min=1e-45) / bound).max()) <= 1
    got = slope_through_backward(z, Activation.Gelu, rows)
    size = cdf + z.double().abs() * density
    assert float(((got - (cdf + z.double() * density)).abs() / size / bound).max()) <= 1


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_16_bit_activations_tails(dtype, rows):
    """Relative to the result: one rounding, and 2^-13 for the short forms of the
    exponential, the reciprocal and Phi.  What these forms flush to zero, below
    2^-126, comes into a result times z, or times its factors in a slope."""
    unit, least = (2.0 ** -11, 2.0 ** -24) if dtype == F16 else (2.0 ** -8, 2.0 ** -126)
    z = torch.linspace(-12.5, 8, 2001, device="cuda").to(dtype)
    zd = z.double()
    cdf, density = normal_cdf_and_density(zd)
    logistic = torch.sigmoid(zd)
    inner = 2 * (2 / torch.pi) ** 0.5 * (zd + 0.044715 * zd ** 3)
    p = torch.sigmoid(inner)
    slope_of_inner = 2 * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * zd ** 2)
    cases = {
        Activation.Gelu: (zd * cdf, [cdf, zd * density]),
        Activation.Silu: (zd * logistic, [logistic, zd * logistic * torch.sigmoid(-zd)]),
        Activation.GeluTanh: (zd * p, [p, zd * p * torch.sigmoid(-inner) * slope_of_inner]),
    }
    for act, (value, terms) in cases.items():
        # the exponential's argument is rounded: 2^-22 of it moves the result
        moved = 2.0 ** -13 + 2.0 ** -22 * inner.abs().clamp(min=1) if act == Activation.GeluTanh else 2.0 ** -13
        got = through_linear(z, act, rows)
        flushed = least + zd.abs() * 2.0 ** -126
        assert bool(((got - value).abs() <= (unit + moved) * value.abs() + flushed).all()), act
        got = slope_through_backward(z, act, rows)
        ref, size = sum(terms), sum(t.abs() for t in terms)
        flushed = least + (1 + zd.abs() * slope_of_inner) * 2.0 ** -126
        assert bool(((got - ref).abs() <= unit * ref.abs() + moved * size + flushed).all()), act


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", list(Activation))
def test_activations_at_the_largest_values(act, dtype, rows):
    """Far out every activation is z or zero and its slope one or zero, exactly, up
    to the type's largest value; infinities and NaN give what the formula gives."""
    top = torch.finfo(dtype).max
    for size in (50.0, 300.0, 6e4, 1e10, 5e19, 1e25, top):
        if size > top:
            continue
        z = torch.tensor([size, -size] * 8, device="cuda").to(dtype)
        value = z.double() if act == Activation.Identity else z.double().clamp(min=0)
        slope = torch.ones_like(value) if act == Activation.Identity else (z > 0).double()
        # silu at -50 is 1e-20 yet, and its slope
        near = 1e-18 if size == 50.0 and act in (Activation.Silu, Activation.Gelu, Activation.GeluTanh) else 0.0
        assert float((through_linear(z, act, rows) - value).abs().max()) <= near, size
        if act != Activation.Identity:
            assert float((slope_through_backward(z, act, rows) - slope).abs().max()) <= near, size
    z = torch.tensor([INF, NAN, -INF] * 5 + [NAN], device="cuda").to(dtype)
    got = ba.linear(torch.zeros((rows, 8), dtype=dtype, device="cuda"),
                    torch.zeros((16, 8), dtype=dtype, device="cuda"), z, activation=act).y[rows - 1]
    assert bool((got[0::3][:5] == INF).all()) and bool(got[1::3].isnan().all())
    below = got[2::3]
    if act == Activation.Identity:
        assert bool((below == -INF).all())
    elif act == Activation.Relu:
        assert bool((below == 0).all())
    else:
        assert bool(below.isnan().all())  # -infinity times zero


# ------------------------------------------------- views that start anywhere
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,inputs,outputs", [(8192, 512, 384), (40000, 64, 128)])
@pytest.mark.parametrize("act", [Activation.Identity, Activation.Silu])
def test_large_views_off_16_bytes(act, rows, inputs, outputs, dtype):
    """Operands whose first value is one past a 16-byte boundary, or whose rows
    are, give what aligned copies of them give, up to the order of sums."""
    def view(width, seed, offset, pitch):
        flat = normal((rows * (width + pitch) + offset,), dtype, seed)
        return flat[offset:].view(rows, width + pitch)[:, :width]

    w, b = normal((outputs, inputs), dtype, 1, 0.1), normal((outputs,), dtype, 2)
    unit = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    for offset, pitch in ((1, 0), (0, 3)):
        x, dy, z = view(inputs, 3, offset, pitch), view(outputs, 4, offset, pitch), view(outputs, 5, offset, pitch)
        xc, dyc, zc = x.clone(), dy.clone(), z.clone()
        for got, want, size in (
                (ba.linear(x, w, b, activation=act).y, ba.linear(xc, w, b, activation=act).y, inputs),
                *zip(vars(ba.linear_backward(dy, x, w, z, activation=act)).values(),
                     vars(ba.linear_backward(dyc, xc, w, zc, activation=act)).values(), (outputs, rows, rows))):
            # two roundings of the result and of dz, and sums of `size` terms of order one
            error = (got.double() - want.double()).norm() / want.double().norm()
            assert float(error) <= 4 * unit + (size ** 0.5 + 16) * 2.0 ** -22


# ------------------------------------------------ a few rows and many outputs
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 4, 7])
def test_few_rows_do_not_depend_on_the_outputs_beside_them(rows, dtype):
    """One output to a warp or four: each is the same sum."""
    x, w = normal((rows, 264), dtype, 1), normal((16001, 264), dtype, 2, 0.1)
    b, res = normal((16001,), dtype, 3), normal((rows, 16001), dtype, 4)
    whole = ba.linear(x, w, b, residual=res, activation=Activation.Silu, save_pre_activation=True)
    for n in (1, 2047, 2049, 3553, 3600, 9473, 16000):
        part = ba.linear(x, w[:n], b[:n], residual=res[:, :n], activation=Activation.Silu,
                         save_pre_activation=True)
        assert torch.equal(part.y, whole.y[:, :n])
        assert torch.equal(part.pre_activation, whole.pre_activation[:, :n])
    ref = x.double() @ w.double().t() + b.double()
    unit = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    size = x.double().abs() @ w.double().abs().t() + b.double().abs()
    bound = unit * ref.abs() + (264 ** 0.5 + 16) * 2.0 ** -22 * size + 2.0 ** -24
    assert bool(((whole.pre_activation.double() - ref).abs() <= bound).all())


# --------------------------------------------------- f32 products' last bits
@pytest.mark.parametrize("inputs", [16, 250, 1000, 4096, 70001])
def test_f32_products_of_one_sign_keep_all_three_parts(inputs):
    """Relative to the sum: 2^-21 for the part products that are left out, 16
    accumulating steps of 2^-23 before sums move to registers, and the roundings
    there.  Without the third parts a product is 2^-16 low in the mean."""
    x, w = uniform((300, inputs), F32, 1, 0.5, 1), uniform((72, inputs), F32, 2, 0.5, 1)
    bound = 2.0 ** -21 + 2.0 ** -19 + (inputs / 256) ** 0.5 * 2.0 ** -24
    ref = x.double() @ w.double().t()
    assert float(((ba.linear(x, w).y.double() - ref).abs() / ref).max()) <= bound
    dy = uniform((300, 72), F32, 3, 0.5, 1)
    ref = dy.double().t() @ x.double()
    assert float(((ba.linear_backward(dy, x, w).weight.double() - ref).abs() / ref).max()) <= bound


# --------------------------------------------------- one output, many rows
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("inputs,outputs", [(40, 1), (1, 40), (1, 1), (300, 1), (1, 300)])
def test_backward_of_one_input_or_output_over_many_rows(inputs, outputs, dtype):
    """A sum of n products in f32 errs by (sqrt(n) + 16) 2^-22 of the terms'
    magnitudes, 16-bit storage rounds dz and the result once each."""
    rows = 100003
    x, w = normal((rows, inputs), dtype, 1), normal((outputs, inputs), dtype, 2)
    dy, z = normal((rows, outputs), dtype, 3), normal((rows, outputs), dtype, 4)
    unit = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    g = ba.linear_backward(dy, x, w, z, activation=Activation.Relu)
    dz = dy.double() * (z > 0).double()
    for got, ref, size, n in (
            (g.x, dz @ w.double(), dz.abs() @ w.double().abs(), outputs),
            (g.weight, dz.t() @ x.double(), dz.abs().t() @ x.double().abs(), rows),
            (g.bias, dz.sum(0), dz.abs().sum(0), rows)):
        bound = unit * ref.abs() + (n ** 0.5 + 16) * 2.0 ** -22 * size + 2.0 ** -24
        assert bool(((got.double() - ref).abs() <= bound).all())
