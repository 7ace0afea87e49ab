"""What the normalised-linear operators are measured on.

The operators are those of a per-particle update block: layer normalisation
of the feature rows and matrix products with bias, activation and residual in
their epilogue, each with its backward pass.  Every case is one pass of one
operator; `run` computes it in plain torch operations in 32 bits, or, when
`own` is set, through the package's public calls.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = ("identity", "relu", "gelu", "gelu_tanh", "silu")
EPS = 1e-5


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _norm(name, op, dtype, rows, dims, pitch=0, affine=True, residual=False):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "dims": dims, "pitch": pitch,
            "affine": affine, "residual": residual}


def _linear(name, op, dtype, rows, inputs, outputs, activation, bias=True, residual=False,
            save=False, pitch=0):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "inputs": inputs,
            "outputs": outputs, "activation": activation, "bias": bias, "residual": residual,
            "save": save, "pitch": pitch}


def listed():
    return [
        # one 4,096-particle rollout's 64 perception features: the latency of one call
        _norm("norm_fwd_rollout", "norm_fwd", "f32", 4096, 64),
        # 1,048,576 particles with 130 features (32 channels, 2D, density gradient): the
        # bandwidth case, rows that are not a multiple of 16 bytes
        _norm("norm_fwd_features", "norm_fwd", "f32", 1048576, 130),
        # the 3D torus rollout's 160 features, backward, parameter gradients over all rows
        _norm("norm_bwd_torus", "norm_bwd", "f32", 16384, 160),
        # the large feature set in bf16, the block's skip gradient added on the way
        _norm("norm_bwd_features", "norm_bwd", "bf16", 1048576, 130, residual=True),
        # wide hidden rows in f16
        _norm("norm_bwd_wide", "norm_bwd", "f16", 16384, 4096),
        # a single row: one particle or pooled readout through a wide layer, bound by the weights
        _linear("linear_fwd_one", "linear_fwd", "bf16", 1, 1024, 4096, "gelu"),
        # the 3D torus update's first layer in f32, its pre-activation kept for training
        _linear("linear_fwd_torus", "linear_fwd", "f32", 16384, 160, 256, "relu", save=True),
        # 256 rollouts of 4,096 particles through the 64 -> 128 layer in bf16
        _linear("linear_fwd_batch", "linear_fwd", "bf16", 1048576, 64, 128, "relu", save=True),
        # a wide layer with its skip connection, bound by the tensor cores
        _linear("linear_fwd_wide", "linear_fwd", "bf16", 8192, 4096, 4096, "gelu_tanh",
                residual=True),
        # the 3D torus update's second layer (35 outputs: an odd width), backward in f32
        _linear("linear_bwd_torus", "linear_bwd", "f32", 16384, 256, 35, "identity"),
        # the batched rollouts' first layer, backward: few weights, a long sum over rows
        _linear("linear_bwd_batch", "linear_bwd", "bf16", 1048576, 64, 128, "relu"),
        # a wide layer's backward in f16
        _linear("linear_bwd_wide", "linear_bwd", "f16", 16384, 1024, 4096, "silu"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over its logarithm; half of them even multiples of eight."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v > 8:
        v = v // 8 * 8
    return min(max(v, lo), hi)


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "linear_fwd", "linear_bwd"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    pitch = rng.choice([0, 0, 0, 1, 8, 24])
    if op.startswith("norm"):
        while True:
            rows, dims = _log_int(rng, 1, 1 << 20), _log_int(rng, 8, 8192)
            if rows * dims <= 1 << 27:
                break
        return _norm(None, op, dtype, rows, dims, pitch, rng.random() < 0.8,
                     op == "norm_bwd" and rng.random() < 0.5)
    while True:
        rows = _log_int(rng, 1, 1 << 20)
        inputs, outputs = _log_int(rng, 8, 4096), _log_int(rng, 8, 4096)
        # f32 costs a plain product several times the 16-bit one's floor
        limit = 1 << (34 if dtype == "f32" else 36)
        if rows * inputs * outputs <= limit and rows * (inputs + outputs) <= 1 << 28:
            break
    return _linear(None, op, dtype, rows, inputs, outputs, rng.choice(ACTIVATIONS),
                   rng.random() < 0.8, op == "linear_fwd" and rng.random() < 0.5,
                   op == "linear_fwd" and rng.random() < 0.5, pitch)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _randn(gen, shape, dtype, scale=1.0, shift=0.0, pitch=0):
    """Normal values; with a pitch, rows of a buffer that is `pitch` elements wider."""
    full = tuple(shape[:-1]) + (shape[-1] + pitch,)
    t = torch.empty(full, dtype=torch.float32, device="cuda")
    t.normal_(shift, scale, generator=gen)
    return t.to(dtype)[..., :shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows, pitch = case["rows"], case["pitch"]
    state = {"case": case}
    if case["op"].startswith("norm"):
        dims = case["dims"]
        # feature rows are not centred: blurred states and gradients carry a mean
        state["x"] = _randn(gen, (rows, dims), dtype, 1.0, 0.5, pitch)
        state["weight"] = _randn(gen, (dims,), dtype, 0.2, 1.0) if case["affine"] else None
        state["bias"] = _randn(gen, (dims,), dtype, 0.2) if case["affine"] else None
        if case["op"] == "norm_bwd":
            state["dy"] = _randn(gen, (rows, dims), dtype, 1.0, 0.0, pitch)
            state["residual_gradient"] = (_randn(gen, (rows, dims), dtype)
                                          if case["residual"] else None)
            var, mean = torch.var_mean(state["x"].float(), dim=-1, correction=0)
            state["mean"], state["rstd"] = mean, torch.rsqrt(var + EPS)
        return state
    inputs, outputs = case["inputs"], case["outputs"]
    # Kaiming-normal weights, as the package's workloads draw them
    state["x"] = _randn(gen, (rows, inputs), dtype, 1.0, 0.0, pitch)
    state["weight"] = _randn(gen, (outputs, inputs), dtype, math.sqrt(2.0 / inputs))
    state["bias"] = _randn(gen, (outputs,), dtype, 0.1) if case["bias"] else None
    if case["op"] == "linear_fwd":
        state["residual"] = (_randn(gen, (rows, outputs), dtype, 1.0, 0.0, pitch)
                             if case["residual"] else None)
        return state
    state["dy"] = _randn(gen, (rows, outputs), dtype, 1.0, 0.0, pitch)
    state["z"] = None
    if case["activation"] != "identity":
        # the pre-activation has the distribution of the forward product's
        state["z"] = _randn(gen, (rows, outputs), dtype, math.sqrt(2.0))
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
    if name == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 3.0 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain_norm_fwd(s):
    x = s["x"].float()
    mean = x.mean(dim=-1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + EPS)
    y = centred * rstd
    if s["weight"] is not None:
        y = y * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _plain_norm_bwd(s):
    dtype = s["x"].dtype
    dy = s["dy"].float()
    xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy if s["weight"] is None else dy * s["weight"].float()
    dx = g - g.mean(dim=-1, keepdim=True) - xhat * (g * xhat).mean(dim=-1, keepdim=True)
    dx = dx * s["rstd"][:, None]
    if s["residual_gradient"] is not None:
        dx = dx + s["residual_gradient"].float()
    out = {"x": dx.to(dtype)}
    if s["weight"] is not None:
        out["weight"] = (dy * xhat).sum(dim=0).to(dtype)
        out["bias"] = dy.sum(dim=0).to(dtype)
    return out


def _plain_linear_fwd(s):
    case, dtype = s["case"], s["x"].dtype
    z = torch.matmul(s["x"].float(), s["weight"].float().t())
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["save"]:
        out["z"] = z.to(dtype)
    return out


def _plain_linear_bwd(s):
    dtype = s["x"].dtype
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_slope(s["z"].float(), s["case"]["activation"])
    out = {"x": torch.matmul(dz, s["weight"].float()).to(dtype),
           "weight": torch.matmul(dz.t(), s["x"].float()).to(dtype)}
    if s["bias"] is not None:
        out["bias"] = dz.sum(dim=0).to(dtype)
    return out


def _own_run(s):
    import burn_automata_b200 as ba

    case = s["case"]
    op = case["op"]
    if op == "norm_fwd":
        r = ba.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        return {"y": r.y, "mean": r.mean, "rstd": r.rstd}
    if op == "norm_bwd":
        g = ba.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"],
                                   residual_gradient=s["residual_gradient"])
        out = {"x": g.x}
        if s["weight"] is not None:
            out["weight"], out["bias"] = g.weight, g.bias
        return out
    act = {"identity": ba.Activation.Identity, "relu": ba.Activation.Relu,
           "gelu": ba.Activation.Gelu, "gelu_tanh": ba.Activation.GeluTanh,
           "silu": ba.Activation.Silu}[case["activation"]]
    if op == "linear_fwd":
        r = ba.linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"],
                      save_pre_activation=case["save"])
        out = {"y": r.y}
        if case["save"]:
            out["z"] = r.pre_activation
        return out
    needs = ("x", "weight", "bias") if case["bias"] else ("x", "weight")
    g = ba.linear_backward(s["dy"], s["x"], s["weight"], pre_activation=s["z"], activation=act,
                           needs=needs)
    out = {"x": g.x, "weight": g.weight}
    if case["bias"]:
        out["bias"] = g.bias
    return out


def run(state):
    if own:
        return _own_run(state)
    return {"norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd,
            "linear_fwd": _plain_linear_fwd,
            "linear_bwd": _plain_linear_bwd}[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# the work a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if case["op"].startswith("norm"):
        dims = case["dims"]
        items = rows * dims
        params = 2 * dims * size if case["affine"] else 0
        if case["op"] == "norm_fwd":
            return {"bytes": 2 * items * size + params + 8 * rows, "flops": 8 * items}
        streams = 3 + (1 if case["residual"] else 0)
        # the weight is read and two gradients written
        params = 3 * dims * size if case["affine"] else 0
        return {"bytes": streams * items * size + params + 8 * rows, "flops": 14 * items}
    inputs, outputs = case["inputs"], case["outputs"]
    weights = inputs * outputs * size
    bias = outputs * size if case["bias"] else 0
    if case["op"] == "linear_fwd":
        streams = 1 + (1 if case["residual"] else 0) + (1 if case["save"] else 0)
        return {"bytes": rows * (inputs + streams * outputs) * size + weights + bias,
                "flops": 2 * rows * inputs * outputs}
    streams = 1 if case["activation"] == "identity" else 2
    return {"bytes": rows * (2 * inputs + streams * outputs) * size + 2 * weights + bias,
            "flops": 4 * rows * inputs * outputs}


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------
def _exact_act(z, name):
    """The activation and its derivative at z (float64)."""
    if name == "identity":
        return z, torch.ones_like(z)
    if name == "relu":
        on = z > 0
        return torch.where(on, z, torch.zeros_like(z)), on.double()
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        # (1 + tanh(u)) / 2 is the logistic function of 2u
        u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(u2)
        slope = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
        return z * p, p + z * p * torch.sigmoid(-u2) * slope
    p = torch.sigmoid(z)
    return z * p, p + z * p * torch.sigmoid(-z)


def _blocks(rows, width):
    """Row ranges of about 2**24 values: 64-bit copies of the whole need not fit at once."""
    step = max(1, (1 << 24) // max(width, 1))
    return [(r, min(r + step, rows)) for r in range(0, rows, step)]


def exact(case, seed):
    s = prepare(case, seed)
    x, rows = s["x"], case["rows"]
    op = case["op"]
    if op == "norm_fwd":
        y = torch.empty((rows, case["dims"]), dtype=torch.float64, device="cuda")
        mean = torch.empty(rows, dtype=torch.float64, device="cuda")
        rstd = torch.empty_like(mean)
        for a, b in _blocks(rows, case["dims"]):
            xb = x[a:b].double()
            m = xb.sum(1) / case["dims"]
            v = ((xb - m[:, None]) ** 2).sum(1) / case["dims"]
            r = 1 / torch.sqrt(v + EPS)
            mean[a:b], rstd[a:b] = m, r
            y[a:b] = (xb - m[:, None]) * r[:, None]
            if s["weight"] is not None:
                y[a:b] = y[a:b] * s["weight"].double() + s["bias"].double()
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "norm_bwd":
        dims = case["dims"]
        dx = torch.empty((rows, dims), dtype=torch.float64, device="cuda")
        dw = torch.zeros(dims, dtype=torch.float64, device="cuda")
        db = torch.zeros_like(dw)
        for a, b in _blocks(rows, dims):
            dy = s["dy"][a:b].double()
            r = s["rstd"][a:b].double()[:, None]
            xh = (x[a:b].double() - s["mean"][a:b].double()[:, None]) * r
            dw += (dy * xh).sum(0)
            db += dy.sum(0)
            g = dy if s["weight"] is None else dy * s["weight"].double()
            part = r * (g - g.sum(1, keepdim=True) / dims
                        - xh * ((g * xh).sum(1, keepdim=True) / dims))
            if s["residual_gradient"] is not None:
                part = part + s["residual_gradient"][a:b].double()
            dx[a:b] = part
        out = {"x": dx}
        if s["weight"] is not None:
            out["weight"], out["bias"] = dw, db
        return out
    inputs, outputs = case["inputs"], case["outputs"]
    w = s["weight"].double()
    if op == "linear_fwd":
        y = torch.empty((rows, outputs), dtype=torch.float64, device="cuda")
        z = torch.empty_like(y) if case["save"] else None
        for a, b in _blocks(rows, inputs + outputs):
            zb = torch.einsum("ri,oi->ro", x[a:b].double(), w)
            if s["bias"] is not None:
                zb = zb + s["bias"].double()
            if z is not None:
                z[a:b] = zb
            yb = _exact_act(zb, case["activation"])[0]
            y[a:b] = yb if s["residual"] is None else yb + s["residual"][a:b].double()
        out = {"y": y}
        if z is not None:
            out["z"] = z
        return out
    dx = torch.empty((rows, inputs), dtype=torch.float64, device="cuda")
    dw = torch.zeros((outputs, inputs), dtype=torch.float64, device="cuda")
    db = torch.zeros(outputs, dtype=torch.float64, device="cuda")
    for a, b in _blocks(rows, inputs + outputs):
        dz = s["dy"][a:b].double()
        if s["z"] is not None:
            dz = dz * _exact_act(s["z"][a:b].double(), case["activation"])[1]
        dx[a:b] = torch.einsum("ro,oi->ri", dz, w)
        dw += torch.einsum("ro,ri->oi", dz, x[a:b].double())
        db += dz.sum(0)
    out = {"x": dx, "weight": dw}
    if s["bias"] is not None:
        out["bias"] = db
    return out
