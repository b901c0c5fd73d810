"""The operators that adapt a trained layer and serve what was adapted, as measurable cases.

A case is a dict of plain values.  ``op`` names the operator and ``train`` its direction (a forward pass, or a forward pass
and the gradients of it):

* ``dropout``       - y = residual + keep * x / (1 - p); ``keep`` comes from a counter-based generator (Philox 4x32, ten
  rounds) and is never stored.  ``shared`` is the axis along which one draw serves all entries (-1: none).
* ``adapter_dense`` - y = act(x W^T + b + scale_g (x D_g^T) U_g^T) + residual, g the adapter of a row's request, and with
  ``gated`` y = value * act(gate), [value | gate] being the argument above.  D_g is [rank, width], U_g [columns, rank].

Inputs of ``dropout`` are ``shape0`` x ``shape1`` x ``width``; those of ``adapter_dense`` are ``requests`` x ``tokens`` x
``width`` with one of ``adapters`` adapters, or none, for each request.  ``out`` is the width of the result.  A training step
returns the gradients of the input and of the adapters, and with ``whole`` those of the shared weight too (it is frozen
otherwise).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _dropout(name, shape, dtype, train, p, shared=-1, residual=False):
    return {"name": name, "op": "dropout", "shape0": shape[0], "shape1": shape[1], "width": shape[2], "dtype": dtype, "train": train,
            "p": p, "shared": shared, "residual": residual}


def _adapter(name, requests, tokens, width, out, dtype, train, adapters, rank, gated=False, activation="none", bias=False, residual=False,
             whole=False):
    return {"name": name, "op": "adapter_dense", "requests": requests, "tokens": tokens, "width": width, "out": out, "dtype": dtype,
            "train": train, "adapters": adapters, "rank": rank, "gated": gated, "activation": activation, "bias": bias,
            "residual": residual, "whole": whole}


def listed():
    return [
        # The update of one token of the single track: nothing but latency.
        _dropout("dropout_token", (1, 1, 384), "bf16", False, 0.25, residual=True),
        # The pair tensor of a 512-token crop in training: one draw for all entries of a column, added to the residual stream.
        _dropout("dropout_pair_512", (512, 512, 128), "bf16", True, 0.25, shared=0, residual=True),
        # A draw for each element of a wide hidden layer.
        _dropout("dropout_hidden", (1, 16384, 2048), "f16", True, 0.1),
        # A 32-bit training run at odd sizes.
        _dropout("dropout_odd", (3, 413, 1001), "f32", True, 0.5, shared=1),
        # One token through the single transition's first half, with the adapter of its request.
        _adapter("adapter_token", 1, 1, 384, 1536, "bf16", False, 8, 16, gated=True, activation="silu"),
        # One token of each of 13 requests through the second half, each with an adapter of its own.
        _adapter("adapter_13_tokens", 13, 1, 1536, 384, "bf16", False, 64, 16, residual=True),
        # A batch of 64 single tokens of different requests through a wide layer.
        _adapter("adapter_64_tokens", 64, 1, 2048, 4096, "bf16", False, 64, 16),
        # The single transition's first half for four complexes of 768 tokens, served together.
        _adapter("adapter_single_4x768", 4, 768, 384, 1536, "bf16", False, 16, 16, gated=True, activation="silu"),
        # The pair transition's first half for eight complexes of 192 tokens, served together.
        _adapter("adapter_pair_8x192", 8, 192 * 192, 128, 512, "bf16", False, 8, 16, gated=True, activation="silu"),
        # An adapter of the pair transition in training on a 384-token crop.
        _adapter("adapter_pair_384", 1, 384 * 384, 128, 512, "bf16", True, 1, 16, gated=True, activation="silu"),
        # A wide layer's adapter in training: the tensor cores and nothing else.
        _adapter("adapter_wide", 1, 8192, 4096, 4096, "bf16", True, 1, 64, activation="gelu_tanh", bias=True, residual=True),
        # Sizes that no tile, vector or alignment divides, several adapters trained at once with the weight that they share.
        _adapter("adapter_odd", 89, 23, 515, 1283, "f16", True, 5, 12, activation="relu", bias=True, whole=True),
    ]


def draw(rng):
    def size(low, high):
        n = math.exp(rng.uniform(math.log(low), math.log(high)))
        # most widths of real layers are multiples of 8 or 64, some are not
        step = rng.choice([1, 1, 8, 64])
        return max(low, round(n / step) * step)

    most = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    op = rng.choice(["dropout", "adapter_dense", "adapter_dense"])
    while True:
        rows = round(math.exp(rng.uniform(0, math.log(512 * 512))))
        train = rng.random() < 0.5
        if op == "dropout":
            first = round(math.exp(rng.uniform(0, math.log(rows)))) if rows > 1 else 1
            case = _dropout("", (first, max(1, rows // first), size(16, 8192)), rng.choice(["bf16", "f16", "f32"]), train,
                            rng.choice([0.1, 0.15, 0.25, 0.5, rng.uniform(0.01, 0.9)]), rng.choice([-1, 0, 1]), rng.random() < 0.5)
        else:
            requests = round(math.exp(rng.uniform(0, math.log(min(rows, 256)))))
            case = _adapter("", requests, max(1, rows // requests), size(16, 4096), size(16, 4096), rng.choice(["bf16", "bf16", "f16"]), train,
                            round(math.exp(rng.uniform(0, math.log(64)))), rng.choice([4, 8, 12, 16, 16, 32, 64, rng.randint(1, 96)]),
                            rng.random() < 0.4, rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]), rng.random() < 0.5,
                            rng.random() < 0.5, rng.random() < 0.3)
            if case["gated"]:
                case["residual"] = False
                if case["activation"] == "none":
                    case["activation"] = "silu"
            if case["requests"] * case["tokens"] * case["adapters"] * case["rank"] > 1 << 28:
                continue  # the plain form's low-rank values of all adapters would not fit the card
        if all(work(case)[m] <= most[m] for m in most):
            del case["name"]
            return case


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "dropout":
        elements = case["shape0"] * case["shape1"] * case["width"]
        moved = 3 if case["residual"] else 2
        return {"bytes": (moved + (2 if case["train"] else 0)) * elements * size, "flops": (4 if case["train"] else 2) * elements}
    rows, width, out, rank = case["requests"] * case["tokens"], case["width"], case["out"], case["rank"]
    columns = 2 * out if case["gated"] else out
    used = min(case["adapters"], case["requests"])
    shared, low = (columns * width + (columns if case["bias"] else 0)) * size, used * rank * (width + columns) * size
    moved = rows * (width + out * (2 if case["residual"] else 1)) * size + shared + low
    if case["train"]:
        moved += rows * (out + width) * size + low + (shared if case["whole"] else 0)
    base = 2 * rows * width * columns
    return {"bytes": moved, "flops": base * (1 + (1 + case["whole"]) * case["train"]) + 2 * rows * rank * (width + columns) * (3 if case["train"] else 1)}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, kind=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).to(kind)

    state = {"case": case}
    if case["op"] == "dropout":
        shape = (case["shape0"], case["shape1"], case["width"])
        state["x"] = normal(*shape)
        state["residual"] = normal(*shape, std=1.5) if case["residual"] else None
        state["seed"], state["sequence"] = 0x9E3779B97F4A7C15 * (seed + 1) % (1 << 63), 7 + seed % 1000
        if case["train"]:
            state["dy"] = normal(*shape, std=0.1)
        return state
    requests, tokens, width, out, rank = (case[k] for k in ("requests", "tokens", "width", "out", "rank"))
    columns, count = 2 * out if case["gated"] else out, case["adapters"]
    state["x"] = normal(requests, tokens, width)
    state["weight"] = normal(columns, width, std=width ** -0.5)
    state["bias"] = normal(columns, std=0.3) if case["bias"] else None
    state["residual"] = normal(requests, tokens, out) if case["residual"] else None
    state["down"] = normal(count, rank, width, std=width ** -0.5)
    state["up"] = normal(count, columns, rank, std=0.3 * rank ** -0.5)
    state["scale"] = torch.rand(count, generator=gen, device="cuda").mul_(1.5).add_(0.5)
    # each request's adapter; of several requests one in ten has none
    index = torch.randint(0, count, (requests,), generator=gen, device="cuda")
    if requests > 1:
        index = torch.where(torch.rand(requests, generator=gen, device="cuda") < 0.1, -1, index)
    state["index"] = index.int()
    if case["train"]:
        state["dy"] = normal(requests, tokens, out, std=0.1)
    return state


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------------------------- the framework's operators


def _run_own(case, s):
    from bionemo_inference_runtime_b200 import ops

    if case["op"] == "dropout":
        shared = None if case["shared"] < 0 else case["shared"]
        out = {"y": ops.dropout(s["x"], case["p"], s["seed"], s["sequence"], residual=s["residual"], shared=shared)}
        if case["train"]:
            out["dx"] = ops.dropout_backward(s["dy"], case["p"], s["seed"], s["sequence"], shared=shared)
        return out
    if case["gated"]:
        forward, backward, more = ops.adapter_gated_dense, ops.adapter_gated_dense_backward, {}
    else:
        forward, backward, more = ops.adapter_dense, ops.adapter_dense_backward, {"residual": s["residual"]}
    given = (s["weight"], s["bias"], s["down"], s["up"], s["index"], s["scale"])
    if not case["train"]:
        return {"y": forward(s["x"], *given, activation=case["activation"], **more)}
    y, saved = forward(s["x"], *given, activation=case["activation"], want_saved=True, **more)
    dx, dweight, dbias, ddown, dup = backward(s["dy"], s["x"], *given, activation=case["activation"], saved=saved,
                                              want_dweight=case["whole"], want_dbias=case["whole"] and case["bias"])
    out = {"y": y, "dx": dx, "ddown": ddown, "dup": dup}
    if case["whole"]:
        out["dweight"] = dweight
        if case["bias"]:
            out["dbias"] = dbias
    return out


# ------------------------------------------------------------------------------------------------- the plain form


def _philox(block, sequence, seed):
    """The four 32-bit words that Philox 4x32-10 makes of a block's number: key the seed, counter (block, sequence)."""
    low = 0xFFFFFFFF
    c = [block & low, block >> 32 & low, torch.full_like(block, sequence & low), torch.full_like(block, sequence >> 32 & low)]
    k = [seed & low, seed >> 32 & low]
    for _ in range(10):
        # (a product of 64 bits; its sign is shifted out)
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32 & low) ^ c[1] ^ k[0], b & low, (a >> 32 & low) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def _keep(case, s):
    """The elements that stay: 16 bits of the generator for each, eight elements to a block, compared with p in steps of 2^-16."""
    shape = [case["shape0"], case["shape1"], case["width"]]
    if case["shared"] >= 0:
        shape[case["shared"]] = 1
    count = math.prod(shape)
    words = torch.stack(_philox(torch.arange((count + 7) // 8, device="cuda"), s["sequence"], s["seed"]), 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:count]
    dropped = round(case["p"] * 65536)
    return (halves >= dropped).view(shape), 65536 / (65536 - dropped) if dropped < 65536 else 0.0


def _activate(z, activation, slope):
    """act(z), and act'(z) where `slope` asks for it."""
    if activation == "none":
        return z, torch.ones_like(z) if slope else None
    if activation == "relu":
        return z.clamp(min=0), (z > 0).float() if slope else None
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
    kind, train = s["x"].dtype, case["train"]
    if case["op"] == "dropout":
        keep, scale = _keep(case, s)
        y = torch.where(keep, s["x"].float() * scale, 0.0)
        out = {"y": (y if s["residual"] is None else y + s["residual"].float()).to(kind)}
        if train:
            out["dx"] = torch.where(keep, s["dy"].float() * scale, 0.0).to(kind)
        return out
    rows, count, rank, n = case["requests"] * case["tokens"], case["adapters"], case["rank"], case["out"]
    x, w = s["x"].float().view(rows, -1), s["weight"].float()
    down, up = s["down"].float().reshape(count * rank, -1), s["up"].float().transpose(1, 2).reshape(count * rank, -1)
    # the low-rank values of all adapters, those of other requests' replaced by zeros
    one = s["index"].view(-1, 1) == torch.arange(count, device="cuda")
    share = (one * s["scale"]).repeat_interleave(case["tokens"], 0).view(rows, count, 1)
    low = ((x @ down.t()).view(rows, count, rank) * share).view(rows, -1)
    z = x @ w.t() + low @ up
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if case["gated"]:
        a, slope = _activate(z[:, n:], case["activation"], train)
        y = z[:, :n] * a
    else:
        a, slope = _activate(z, case["activation"], train)
        y = a if s["residual"] is None else a + s["residual"].float().view(rows, -1)
    out = {"y": y.to(kind).view(*s["x"].shape[:2], n)}
    if train:
        dy = s["dy"].float().view(rows, n)
        dz = torch.cat([dy * a, dy * z[:, :n] * slope], 1) if case["gated"] else dy * slope
        dlow = ((dz @ up.t()).view(rows, count, rank) * share).view(rows, -1)
        out["dx"] = (dz @ w + dlow @ down).to(kind).view(s["x"].shape)
        out["ddown"] = (dlow.t() @ x).to(kind).view(s["down"].shape)
        out["dup"] = (low.t() @ dz).to(kind).view(count, rank, -1).transpose(1, 2).contiguous()
        if case["whole"]:
            out["dweight"] = (dz.t() @ x).to(kind)
            if s["bias"] is not None:
                out["dbias"] = dz.sum(0).to(kind)
    return out


def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


# -------------------------------------------------------------------------------------- the definition, in 64 bits


def _exact_dropout(case, s):
    """Philox by products of 16-bit halves, element by element of the tensor's own coordinates."""
    sizes = [case["shape0"], case["shape1"], case["width"]]
    at = torch.meshgrid(*(torch.arange(n, device="cuda") for n in sizes), indexing="ij")
    number = torch.zeros_like(at[0])
    for axis, n in enumerate(sizes):
        if axis != case["shared"]:
            number = number * n + at[axis]
    del at

    def product(a, m):  # (high, low) words of a * m
        low, high = (a & 0xFFFF) * m, (a >> 16) * m  # both below 2^48
        total = low + ((high & 0xFFFF) << 16)
        return (high >> 16) + (total >> 32), total & 0xFFFFFFFF

    block, place = number // 8, number % 8
    c0, c1 = block % (1 << 32), block // (1 << 32)
    c2, c3 = (torch.full_like(block, w) for w in (s["sequence"] % (1 << 32), s["sequence"] // (1 << 32)))
    k0, k1 = s["seed"] % (1 << 32), s["seed"] // (1 << 32)
    for r in range(10):
        (h0, l0), (h1, l1) = product(c0, 0xD2511F53), product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ (k0 + r * 0x9E3779B9) % (1 << 32), l1, h0 ^ c3 ^ (k1 + r * 0xBB67AE85) % (1 << 32), l0
    word = torch.where(place < 2, c0, torch.where(place < 4, c1, torch.where(place < 6, c2, c3)))
    value = torch.where(place % 2 == 0, word % (1 << 16), word // (1 << 16))
    dropped = round(case["p"] * 65536)
    factor = torch.where(value < dropped, 0.0, 1.0).double() / (1 - dropped / 65536)
    out = {"y": s["x"] * factor + (0 if s["residual"] is None else s["residual"])}
    if case["train"]:
        out["dx"] = s["dy"] * factor
    return out


def exact(case, seed):
    """The definitions in float64; the gradients are those of automatic differentiation."""
    F = torch.nn.functional
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    if case["op"] == "dropout":
        return _exact_dropout(case, s)
    acts = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}
    names = ["x", "down", "up"] + (["weight"] + (["bias"] if case["bias"] else []) if case["whole"] else [])
    for name in names:
        s[name].requires_grad_(case["train"])
    with torch.set_grad_enabled(case["train"]):
        z = F.linear(s["x"], s["weight"], s["bias"])
        for g in range(case["adapters"]):
            of = (s["index"] == g).nonzero().view(-1)
            if of.numel():
                z = z.index_add(0, of, s["scale"][g] * F.linear(F.linear(s["x"][of], s["down"][g]), s["up"][g]))
        if case["gated"]:
            value, gate = z.chunk(2, -1)
            y = value * acts[case["activation"]](gate)
        else:
            y = acts[case["activation"]](z)
            y = y if s["residual"] is None else y + s["residual"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [s[name] for name in names], s["dy"], allow_unused=True)  # (no request may have an adapter)
        out |= {"d" + name: torch.zeros_like(s[name]) if g is None else g for name, g in zip(names, grads)}
    return out
