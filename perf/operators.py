"""The operators that train and serve a transition, as measurable cases.

A case is a dict of plain values.  ``op`` names the operator and ``train`` its direction (a forward pass, or a forward
pass and the gradients of it):

* ``layer_norm``  - y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis.
* ``gated_dense`` - y = value * act(gate), [value | gate] = x W^T + b; W holds the value rows, then the gate rows.
* ``dense``       - y = act(x W^T + b) + residual.

``rows`` x ``width`` is the input, ``out`` the width of the result, ``dtype`` the type of the activations and (but for
``layer_norm`` with ``f32_weights``) of the parameters and their gradients.
"""

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _norm(name, rows, width, dtype, train, f32_weights=False):
    return {"name": name, "op": "layer_norm", "rows": rows, "width": width, "out": width, "dtype": dtype, "train": train,
            "f32_weights": f32_weights}


def _gated(name, rows, width, out, dtype, train, activation="silu", bias=False):
    return {"name": name, "op": "gated_dense", "rows": rows, "width": width, "out": out, "dtype": dtype, "train": train,
            "activation": activation, "bias": bias}


def _dense(name, rows, width, out, dtype, train, activation="none", bias=False, residual=False):
    return {"name": name, "op": "dense", "rows": rows, "width": width, "out": out, "dtype": dtype, "train": train,
            "activation": activation, "bias": bias, "residual": residual}


def listed():
    return [
        # One token of the single track: nothing but latency.
        _norm("layer_norm_token", 1, 384, "bf16", False),
        # The pair tensor of a 512-token crop in training, parameters kept in 32 bits.
        _norm("layer_norm_pair_512", 512 * 512, 128, "bf16", True, f32_weights=True),
        # A 32-bit training run at an odd width and row count.
        _norm("layer_norm_odd", 1237, 1001, "f32", True),
        # The widest rows.
        _norm("layer_norm_wide", 6001, 8192, "f16", False),
        # One token through the single transition's first half.
        _gated("gated_token", 1, 384, 1536, "bf16", False),
        # The single transition's first half for a 768-token complex.
        _gated("gated_single_768", 768, 384, 1536, "bf16", False),
        # The pair transition's first half for a 384-token crop in training.
        _gated("gated_pair_384", 384 * 384, 128, 512, "bf16", True),
        # A wider gated block with biases in half precision, a ragged number of rows.
        _gated("gated_gelu", 5003, 768, 3072, "f16", True, activation="gelu", bias=True),
        # A few tokens through the single transition's second half.
        _dense("dense_tokens", 3, 1536, 384, "bf16", False, residual=True),
        # The pair transition's second half with its residual at 512 tokens.
        _dense("dense_pair_512", 512 * 512, 512, 128, "bf16", False, residual=True),
        # A wide layer in training: the tensor cores and nothing else.
        _dense("dense_wide", 8192, 4096, 4096, "bf16", True, activation="gelu_tanh", bias=True, residual=True),
        # Sizes that no tile, vector or alignment divides.
        _dense("dense_odd", 2047, 515, 1283, "bf16", True, activation="relu", bias=True),
    ]


def draw(rng):
    def size(low, high):
        n = math.exp(rng.uniform(math.log(low), math.log(high)))
        # most widths of real layers are multiples of 8 or 64, some are not
        step = rng.choice([1, 1, 8, 64])
        return max(low, round(n / step) * step)

    most = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    op = rng.choice(["layer_norm", "gated_dense", "dense"])
    while True:
        rows = round(math.exp(rng.uniform(0, math.log(512 * 512))))
        train = rng.random() < 0.6
        dtype = rng.choice(["bf16", "bf16", "f16"])
        if op == "layer_norm":
            case = _norm("", rows, size(16, 8192), rng.choice(["bf16", "f16", "f32"]), train, rng.random() < 0.5)
        elif op == "gated_dense":
            case = _gated("", rows, size(16, 2048), size(16, 8192), dtype, train, rng.choice(["silu", "gelu", "gelu_tanh", "sigmoid", "relu"]),
                          rng.random() < 0.5)
        else:
            case = _dense("", rows, size(16, 4096), size(16, 4096), dtype, train, rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]),
                          rng.random() < 0.5, rng.random() < 0.5)
        if all(work(case)[m] <= most[m] for m in most):
            del case["name"]
            return case


def work(case):
    rows, width, out = case["rows"], case["width"], case["out"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "layer_norm":
        params = 2 * width * (4 if case["f32_weights"] else size)
        passes = 4 if case["train"] else 2  # x and y; dy and dx
        return {"bytes": passes * rows * width * size + (2 if case["train"] else 1) * params,
                "flops": (19 if case["train"] else 8) * rows * width}
    columns = 2 * out if case["op"] == "gated_dense" else out
    params = (columns * width + (columns if case["bias"] else 0)) * size
    moved = rows * (width + out * (2 if case.get("residual") else 1)) * size + params
    if case["train"]:
        moved += rows * (out + width) * size + params
    return {"bytes": moved, "flops": (6 if case["train"] else 2) * rows * width * columns}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, width, out, dtype = case["rows"], case["width"], case["out"], DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, kind=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).add_(mean).to(kind)

    state = {"case": case}
    if case["op"] == "layer_norm":
        kind = torch.float32 if case["f32_weights"] else dtype
        # a residual stream: rows with a mean and a spread of their own
        state["x"] = normal(rows, width, std=1.5, mean=0.25)
        state["weight"], state["bias"] = normal(width, std=0.2, mean=1.0, kind=kind), normal(width, std=0.1, kind=kind)
    else:
        columns = 2 * out if case["op"] == "gated_dense" else out
        state["x"] = normal(rows, width)
        state["weight"] = normal(columns, width, std=width ** -0.5)
        state["bias"] = normal(columns, std=0.3) if case["bias"] else None
        state["residual"] = normal(rows, out) if case.get("residual") else None
    if case["train"]:
        state["dy"] = normal(rows, out, std=0.1)
    return state


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------------------------- the framework's operators


def _run_own(case, s):
    from bionemo_inference_runtime_b200 import ops

    if case["op"] == "layer_norm":
        if not case["train"]:
            return {"y": ops.layer_norm(s["x"], s["weight"], s["bias"], EPS)}
        y, stats = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS, want_stats=True)
        dx, dweight, dbias = ops.layer_norm_backward(s["dy"], s["x"], stats, s["weight"])
        return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
    if case["op"] == "gated_dense":
        forward, backward, more = ops.gated_dense, ops.gated_dense_backward, {}
    else:
        forward, backward, more = ops.dense, ops.dense_backward, {"residual": s["residual"]}
    if not case["train"]:
        return {"y": forward(s["x"], s["weight"], s["bias"], activation=case["activation"], **more)}
    y, saved = forward(s["x"], s["weight"], s["bias"], activation=case["activation"], want_saved=True, **more)
    dx, dweight, dbias = backward(s["dy"], s["x"], s["weight"], s["bias"], activation=case["activation"], saved=saved)
    return {"y": y, "dx": dx, "dweight": dweight} | ({"dbias": dbias} if case["bias"] else {})


# ------------------------------------------------------------------------------------------------- the plain form


def _activate(z, activation, slope):
    """act(z), and act'(z) where `slope` asks for it."""
    if activation == "none":
        return z, torch.ones_like(z) if slope else None
    if activation == "relu":
        return z.clamp(min=0), (z > 0).float() if slope else None
    if activation == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s, s * (1 - s) if slope else None
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s)) if slope else None
    if activation == "gelu":
        p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5 if slope else None
    c = (2 / math.pi) ** 0.5  # gelu_tanh
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z) if slope else None


def _run_plain(case, s):
    x, w, kind = s["x"].float(), s["weight"].float(), s["x"].dtype
    bias = None if s["bias"] is None else s["bias"].float()
    train = case["train"]
    if case["op"] == "layer_norm":
        centred = x - x.mean(-1, keepdim=True)
        rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
        normed = centred * rstd
        out = {"y": (normed * w + bias).to(kind)}
        if train:
            dy = s["dy"].float()
            g = dy * w
            dx = rstd * (g - g.mean(-1, keepdim=True) - normed * (g * normed).mean(-1, keepdim=True))
            out |= {"dx": dx.to(kind), "dweight": (dy * normed).sum(0).to(s["weight"].dtype), "dbias": dy.sum(0).to(s["weight"].dtype)}
        return out
    z = x @ w.t()
    if bias is not None:
        z = z + bias
    if case["op"] == "gated_dense":
        value, gate = z[:, :case["out"]], z[:, case["out"]:]
        a, slope = _activate(gate, case["activation"], train)
        out = {"y": (value * a).to(kind)}
        if train:
            dy = s["dy"].float()
            dz = torch.cat([dy * a, dy * value * slope], 1)
    else:
        a, slope = _activate(z, case["activation"], train)
        out = {"y": (a if s["residual"] is None else a + s["residual"].float()).to(kind)}
        if train:
            dz = s["dy"].float() * slope
    if train:
        out |= {"dx": (dz @ w).to(kind), "dweight": (dz.t() @ x).to(kind)}
        if bias is not None:
            out["dbias"] = dz.sum(0).to(kind)
    return out


def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


# -------------------------------------------------------------------------------------- the definition, in 64 bits


def exact(case, seed):
    """The definitions in float64; the gradients are those of automatic differentiation."""
    F = torch.nn.functional
    acts = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "sigmoid": torch.sigmoid, "gelu": F.gelu,
            "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}
    s = {k: v.double() if torch.is_tensor(v) else v for k, v in _inputs(case, seed).items()}
    leaves = [t.requires_grad_(case["train"]) for t in (s["x"], s["weight"], s["bias"]) if t is not None]
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "layer_norm":
            y = F.layer_norm(s["x"], (case["width"],), s["weight"], s["bias"], EPS)
        elif case["op"] == "gated_dense":
            value, gate = F.linear(s["x"], s["weight"], s["bias"]).chunk(2, -1)
            y = value * acts[case["activation"]](gate)
        else:
            y = acts[case["activation"]](F.linear(s["x"], s["weight"], s["bias"]))
            y = y if s["residual"] is None else y + s["residual"]
    out = {"y": y.detach()}
    if case["train"]:
        out |= dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, s["dy"])))
    return out
