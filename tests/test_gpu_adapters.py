"""Dense layers with low-rank adapters against the formulas in 64 bits.

Tolerances are bounds derived from what is rounded, with u half the spacing of the type: sums in 32 bits are off by 2^-18 of their absolute
terms (up to a few thousand), the low-rank values t and their gradients dt, held as two numbers of the type, by u^2 of theirs (and half of
the smallest number, where the second one is that small), the gradient before the activation by u where it goes from one kernel to the
next, every result by u.  Slopes are at most 1.2, the second derivatives 0.8.
"""

import math

import pytest
import torch

import bionemo_inference_runtime_b200 as b200
from bionemo_inference_runtime_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM = 2.0 ** -18
ACTS = {
    "none": lambda t: t,
    "relu": lambda t: t.clamp(min=0),
    "silu": lambda t: t / (1 + torch.exp(-t)),
    "gelu": lambda t: 0.5 * t * (1 + torch.erf(t / math.sqrt(2))),
    "gelu_tanh": lambda t: 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))),
    "sigmoid": lambda t: 1 / (1 + torch.exp(-t)),
}


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    _lib.reset_device_status()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def randn(*shape, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def within(got, want, bound, what):
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = (got.double() - want).abs() - bound
    worst = excess.max().item() if excess.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} over its bound (at most {bound.max().item():.3g})"


def layer(rows, K, N, count, rank, dtype=torch.bfloat16, gated=False, bias=True, residual=True, index=None, seed=0):
    columns = 2 * N if gated else N
    g = torch.Generator(device=DEV).manual_seed(seed + 9)
    return {
        "x": randn(rows, K, seed=seed + 1, dtype=dtype), "w": randn(columns, K, seed=seed + 2, dtype=dtype, std=K ** -0.5),
        "bias": randn(columns, seed=seed + 3, dtype=dtype, std=0.3) if bias else None,
        "residual": randn(rows, N, seed=seed + 4, dtype=dtype) if residual and not gated else None,
        "down": randn(count, rank, K, seed=seed + 5, dtype=dtype, std=K ** -0.5),
        "up": randn(count, columns, rank, seed=seed + 6, dtype=dtype, std=0.5 * rank ** -0.5),
        "scale": torch.rand(count, generator=g, device=DEV) * 1.5 + 0.25, "index": index, "gated": gated,
        "dy": randn(rows, N, seed=seed + 7, dtype=dtype, std=0.1),
    }


def requests(count, of, seed=0, kind=torch.int32):
    """Adapters of `of` requests, some of them none."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    index = torch.randint(-1, count, (of,), generator=g, device=DEV)
    return index.to(kind)


def check(x, w, bias, residual, down, up, scale, index, gated, dy, activation="none", backward=True, whole=True):
    """Forward and backward of x [rows, K] (with an index of n entries: [n, rows / n, K])."""
    rows, K = x.shape
    N = dy.shape[1]
    u, tiny = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal
    least = torch.finfo(x.dtype).tiny * u  # half of the smallest number
    lead = (rows,) if index is None else (index.numel(), rows // index.numel())
    shaped = lambda t: None if t is None else t.view(*lead, -1)  # noqa: E731
    forward, back, more = (ops.adapter_gated_dense, ops.adapter_gated_dense_backward, {}) if gated else (
        ops.adapter_dense, ops.adapter_dense_backward, {"residual": shaped(residual)})
    given = (w, bias, down, up, index, scale)
    y, saved = forward(shaped(x), *given, activation=activation, want_saved=True, **more)
    again = forward(shaped(x), *given, activation=activation, **more)
    assert torch.equal(y, again)  # whether values are kept or not

    of = torch.zeros(rows, dtype=torch.long, device=DEV) if index is None else index.long().repeat_interleave(rows // index.numel())
    has = [(of == g).nonzero().view(-1) for g in range(down.shape[0])]
    xd, wd, dd, ud = x.double(), w.double(), down.double(), up.double()
    z = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    t = xd.new_zeros(rows, down.shape[1])
    t_off = torch.zeros_like(t)
    z_off = torch.zeros_like(z)
    for g, r in enumerate(has):
        s = float(scale[g])
        t[r] = s * (xd[r] @ dd[g].t())
        sums = s * (xd[r].abs() @ dd[g].abs().t())
        t_off[r] = SUM * sums + 1.01 * u * u * t[r].abs() + least
        z[r] += t[r] @ ud[g].t()
        size[r] += sums @ ud[g].abs().t()
        z_off[r] = t_off[r] @ ud[g].abs().t()
    z_off = z_off + SUM * size
    pre = (z[:, N:] if gated else z).clone().requires_grad_(True)
    with torch.enable_grad():
        a = ACTS[activation](pre)
        slope = torch.autograd.grad(a.sum(), pre)[0]
    a = a.detach()
    if gated:
        value, off_v, off_g = z[:, :N], z_off[:, :N], z_off[:, N:]
        want, off = value * a, 1.02 * (a.abs() * off_v + value.abs() * 1.2 * off_g)
    else:
        want, off = a, 1.2 * z_off
        if residual is not None:
            want, off = want + residual.double(), off + SUM * residual.double().abs()
    within(y.view(rows, N), want, 1.01 * u * want.abs() + off + tiny, "y")
    if not backward:
        return
    # with the values before the activation kept, where they are, and computed again
    for kept in (saved,) if saved[1] is None else (saved, (saved[0], None)):
        got = back(shaped(dy), shaped(x), *given, activation=activation, saved=kept, want_dweight=whole, want_dbias=whole and bias is not None)
        d = dy.double()
        if gated:
            dz = torch.cat([d * a, d * value * slope], 1)
            off = torch.cat([1.2 * d.abs() * off_g, 1.02 * d.abs() * (1.2 * off_v + 0.8 * value.abs() * off_g)], 1)
        else:
            dz, off = d * slope, 0.8 * d.abs() * z_off
        if activation == "relu":  # its slope jumps: where the sum may have the other sign, either is right
            near = pre.detach().abs() <= (z_off[:, N:] if gated else z_off)
            jump = near * d.abs() * (value.abs() if gated else 1)
            off = off + (torch.cat([near * d.abs() * z_off[:, N:], jump], 1) if gated else jump)
        off_low = off  # of dz for the adapters' gradients: in two terms where rows are few
        if activation != "none" or gated:
            off = off + 1.01 * u * dz.abs() + tiny
            off_low = off_low + 1.01 * u * u * dz.abs() + least if kept[1] is not None and rows <= 512 and rows * min(down.shape[1], dz.shape[1]) <= 4096 else off
        dx, dx_off = dz @ wd, off @ wd.abs() + SUM * (dz.abs() @ wd.abs())
        ddown, ddown_off, dup, dup_off = torch.zeros_like(dd), torch.zeros_like(dd), torch.zeros_like(ud), torch.zeros_like(ud)
        for g, r in enumerate(has):
            s = float(scale[g])
            dt = s * (dz[r] @ ud[g])
            sums = s * (dz[r].abs() @ ud[g].abs())
            dt_off = s * (off_low[r] @ ud[g].abs()) + SUM * sums + 1.01 * u * u * dt.abs() + least
            dx[r] += dt @ dd[g]
            dx_off[r] += dt_off @ dd[g].abs() + SUM * (sums @ dd[g].abs())
            ddown[g] = dt.t() @ xd[r]
            ddown_off[g] = dt_off.t() @ xd[r].abs() + SUM * (dt.abs().t() @ xd[r].abs())
            dup[g] = dz[r].t() @ t[r]
            dup_off[g] = off_low[r].t() @ (t[r].abs() + t_off[r]) + dz[r].abs().t() @ t_off[r] + SUM * (dz[r].abs().t() @ t[r].abs())
        wanted = [("dx", got[0].view(rows, K), dx, dx_off), ("ddown", got[3], ddown, ddown_off), ("dup", got[4], dup, dup_off)]
        if whole:
            wanted.append(("dweight", got[1], dz.t() @ xd, off.t() @ xd.abs() + SUM * (dz.abs().t() @ xd.abs())))
            if bias is not None:
                wanted.append(("dbias", got[2], dz.sum(0), off.sum(0) + SUM * dz.abs().sum(0)))
        for name, have, want, bound in wanted:
            within(have, want, 1.01 * u * want.abs() + bound + tiny, name)


# rows around a block's own values (8), the few rows (16, 64), the kernels by 32 rows and the tiles of 128 and 256
SIZES = [(1, 1, 1, 1), (1, 384, 96, 16), (2, 8, 8, 3), (5, 64, 33, 12), (8, 100, 130, 8), (9, 256, 64, 8), (17, 40, 24, 17), (33, 64, 72, 16), (64, 96, 40, 32),
         (65, 128, 128, 16), (100, 515, 129, 7), (129, 72, 65, 33), (200, 128, 257, 16), (300, 384, 200, 64), (513, 64, 512, 5), (700, 130, 133, 40),
         (1000, 96, 320, 16), (2500, 520, 136, 24), (333, 1000, 1, 100), (600, 1541, 70, 256)]


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows,K,N,rank", SIZES)
def test_one_adapter(rows, K, N, rank, gated):
    more = (rows + K + N) % 2 == 0
    dtype = torch.float16 if (rows + N) % 3 == 0 else torch.bfloat16
    check(activation="silu", **layer(rows, K, N, 1, rank, dtype, gated, more, not more))


# (requests, rows of each): single tokens, rows that no tile divides, whole tiles, more rows than run at once
BATCHES = [(1, 1), (7, 1), (16, 1), (40, 1), (64, 1), (65, 1), (300, 1), (4200, 1), (13, 3), (89, 23), (5, 64), (9, 128), (3, 100), (4, 256), (2, 700),
           (6, 3000), (700, 31)]


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("n,each", BATCHES)
def test_adapters_of_many_requests(n, each, gated):
    kind = torch.int64 if n % 2 else torch.int32
    count, rank = min(n, 37) + 2, 16 if each % 2 else 20
    check(activation="gelu", **layer(n * each, 136, 72, count, rank, torch.bfloat16, gated, True, True, requests(count, n, kind=kind)))


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("activation", list(ACTS))
@pytest.mark.parametrize("rows,K", [(6, 64), (50, 64), (150, 64), (150, 1544)])
def test_activations(rows, K, activation, gated):
    """Few rows, tiles of rows, few inputs and many."""
    for dtype in (torch.bfloat16, torch.float16):
        check(activation=activation, **layer(rows, K, 72, 3, 16, dtype, gated, True, True, requests(3, rows // 2)))


@pytest.mark.parametrize("rows,K,N,gated,index", [(147456, 128, 512, True, [1]), (40001, 128, 512, False, [0]), (30011, 512, 128, False, None),
                                                  (120000, 72, 200, True, [1, -1, 0]), (270000, 16, 1024, True, [0, 1, 1])])
def test_many_rows(rows, K, N, gated, index):
    """The last has so many that the backward pass takes them in several chunks."""
    index = None if index is None else torch.tensor(index, device=DEV)
    check(activation="silu", whole=False, **layer(rows, K, N, 1 if index is None else 2, 16, torch.bfloat16, gated, False, False, index))


def test_entries_that_are_no_adapter():
    given = layer(600, 64, 48, 4, 8, index=torch.tensor([0, -1, 4, 3, 2 ** 31 - 1, -2 ** 31], device=DEV, dtype=torch.int32))
    check(**given)
    given["index"] = torch.tensor([2, -(2 ** 40), 2 ** 40, 2 ** 32, 3, 2 ** 63 - 1], device=DEV)
    check(**given)
    for n in (5, 40, 600):  # none at all
        none = layer(n, 64, 48, 4, 8, index=torch.full((n,), -1, device=DEV))
        check(**none)
        y = ops.adapter_dense(none["x"], none["w"], none["bias"], none["down"] * math.nan, none["up"] * math.inf, none["index"], none["scale"])
        assert torch.isfinite(y).all()


@pytest.mark.parametrize("n,each", [(6, 1), (48, 1), (200, 1), (12, 40), (6, 256), (40, 100)])
@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
def test_nothing_of_a_request_reaches_another(n, each, gated):
    """NaN and infinities in the rows of two requests and in the weights of an adapter stay with them, forward and backward."""
    index = torch.arange(n, device=DEV, dtype=torch.int32) % 4
    index[1] = -1
    given = layer(n * each, 72, 40, 4, 12, gated=gated, residual=False, index=index)
    forward, back = (ops.adapter_gated_dense, ops.adapter_gated_dense_backward) if gated else (ops.adapter_dense, ops.adapter_dense_backward)

    def run(x, down, up, dy):
        layers = (given["w"], given["bias"], down, up, index, given["scale"])
        y, saved = forward(x, *layers, activation="silu", want_saved=True)
        return [y, *back(dy, x, *layers, activation="silu", saved=saved)]

    x, dy = given["x"].view(n, each, -1), given["dy"].view(n, each, -1)
    clean = run(x, given["down"], given["up"], dy)
    bad_x, bad_down, bad_up = x.clone(), given["down"].clone(), given["up"].clone()
    bad_x[1], bad_x[2, 0, 3], bad_down[3, 0, 5], bad_up[3, 7, 1] = math.nan, math.inf, math.nan, math.inf
    bad = run(bad_x, bad_down, bad_up, dy)
    rest = (index != 3).nonzero().view(-1)
    rest = rest[(rest != 1) & (rest != 2)]
    assert torch.equal(bad[0][rest], clean[0][rest]) and torch.equal(bad[1][rest], clean[1][rest])
    for k in (4, 5):  # adapters 0 and 1 have neither of these rows (row 1 has none, row 2 is adapter 2's)
        assert torch.equal(bad[k][:2], clean[k][:2])
    again = run(x, given["down"], given["up"], dy)
    assert all(a is None if c is None else torch.equal(a, c) for a, c in zip(again, clean, strict=True))  # the same bits each time


@pytest.mark.parametrize("rows", [2, 40, 300, 700])
def test_what_leaves_the_range_of_16_bits_is_infinite(rows):
    """A low-rank value past 65504 in fp16 is an infinity there, not the NaN of what it lacks."""
    given = layer(rows, 64, 40, 1, 8, torch.float16, residual=False, bias=False)
    x = given["x"].abs() * 100
    y = ops.adapter_dense(x, given["w"], None, given["down"].abs() + 20, given["up"].abs() + 0.01)
    assert torch.isinf(y).all() and (y > 0).all()


def test_strides():
    """Operands that no aligned load takes as they lie: odd pitches, transposed, broadcast and single-column tensors."""
    for n, each in ((6, 1), (60, 1), (10, 40)):
        index = requests(3, n)
        base = randn(n, each, 167, seed=1)
        for x in (base[..., 3:103], base[..., :100:2], base.transpose(0, 1)[:, :n].transpose(0, 1)[..., 1:90], base[:, :1].expand(n, each, 167), base[..., :1]):
            K = x.shape[-1]
            given = layer(n * each, K, 56, 3, 13, index=index, residual=False, bias=False)
            w = given["w"].t().contiguous().t()
            down = torch.cat([given["down"], given["down"]], 2)[..., :K]
            up = given["up"].transpose(1, 2).contiguous().transpose(1, 2)
            dy = randn(n, each, 59, seed=2)[..., 2:58]
            y, saved = ops.adapter_dense(x, w, None, down, up, index.long(), given["scale"], want_saved=True)
            want, kept = ops.adapter_dense(x.contiguous(), given["w"], None, given["down"], given["up"], index, given["scale"], want_saved=True)
            u = 2.0 ** -8
            near = 2.02 * u * want.abs() + 2.0 ** -9  # (another order of the same sums, each rounded once)
            assert ((y.float() - want.float()).abs() <= near).all()
            got = ops.adapter_dense_backward(dy, x, w, None, down, up, index, given["scale"], saved=saved)
            plain = ops.adapter_dense_backward(dy.contiguous(), x.contiguous(), given["w"], None, given["down"], given["up"], index, given["scale"], saved=kept)
            for a, b in zip(got, plain, strict=True):
                assert a is None and b is None or ((a.double() - b.double()).norm() <= 4 * u * b.double().norm() + 1e-6)


@pytest.mark.parametrize("rows,K,N,count,rank,n", [(3, 64, 40, 2, 8, 3), (40, 64, 40, 3, 16, 40), (200, 72, 136, 2, 12, 4), (521, 64, 40, 1, 20, 1), (1311, 40, 520, 5, 16, 19),
                                                   (9479, 128, 64, 1, 16, 1)])
@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("kept", [0, 1])
def test_nothing_is_written_behind_the_results(rows, K, N, count, rank, n, gated, kept):
    """Through the C entry points, with canaries behind y, the low-rank values, every gradient and the workspace."""
    index = requests(count, n)
    given = layer(rows, K, N, count, rank, gated=bool(gated), residual=False, bias=False, index=index)
    columns, act = N * (1 + gated), _act("silu")
    lib = _lib.load()

    def held(n_bytes):
        return torch.full((n_bytes + (1 << 18),), 0x5A, dtype=torch.uint8, device=DEV)

    pad = lambda t: torch.nn.functional.pad(t, (0, -t.shape[-1] % 8))  # noqa: E731
    up, down = pad(given["up"]).contiguous(), pad(given["down"]).contiguous()

    class Adapters(_lib.ctypes.Structure):
        _fields_ = [("down", _lib.c_void_p), ("up", _lib.c_void_p), ("ds", _lib.c_int64), ("us", _lib.c_int64), ("scale", _lib.c_void_p),
                    ("scale_all", _lib.c_float), ("index", _lib.c_void_p), ("bytes", _lib.c_int), ("per", _lib.c_int64), ("count", _lib.c_int), ("rank", _lib.c_int)]

    a = Adapters(down.data_ptr(), up.data_ptr(), down.shape[-1], up.shape[-1], given["scale"].data_ptr(), 1.0, index.data_ptr(), 4, rows // n, count, rank)
    stream = torch.cuda.current_stream().cuda_stream
    sizes = {"y": rows * N * 2, "low": rows * lib.b200ta_adapter_low_bytes(rank), "dx": rows * K * 2, "ddown": count * rank * K * 2, "dup": count * columns * rank * 2}
    need = lib.b200ta_adapter_dense_backward_workspace_bytes(act, gated, kept, 0, _lib.ctypes.byref(a), rows, K, N)
    sizes["workspace"] = need
    pitch = (N + 7) // 8 * 8 * (1 + gated)
    sizes["saved"] = rows // n * n * pitch * 4
    got = {k: held(v) for k, v in sizes.items()}
    x, w, dy = given["x"], given["w"], given["dy"]
    rows = rows // n * n
    saved = got["saved"].data_ptr() if kept else None
    _lib.call("b200ta_adapter_dense", x.data_ptr(), K, w.data_ptr(), K, None, None, 0, got["y"].data_ptr(), N, saved, pitch, _lib.ctypes.byref(a),
              got["low"].data_ptr(), 0, act, gated, rows, K, N, stream)
    _lib.call("b200ta_adapter_dense_backward", dy.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, None, saved, pitch, _lib.ctypes.byref(a),
              got["low"].data_ptr(), got["dx"].data_ptr(), K, None, None, got["ddown"].data_ptr(), got["dup"].data_ptr(), got["workspace"].data_ptr(), need, 0,
              act, gated, rows, K, N, stream)
    torch.cuda.synchronize()
    used = {"y": rows * N * 2, "low": rows * lib.b200ta_adapter_low_bytes(rank), "dx": rows * K * 2}
    for name, t in got.items():
        assert (t[used.get(name, sizes[name]):] == 0x5A).all(), name


def _act(name):
    return ops.ACTIVATIONS[name]


def test_out():
    for n in (3, 40, 300):
        given = layer(n, 64, 40, 3, 8, index=requests(3, n))
        args = (given["w"], given["bias"], given["down"], given["up"], given["index"], given["scale"])
        want = ops.adapter_dense(given["x"], *args, residual=given["residual"])
        held = torch.zeros(n, 56, device=DEV, dtype=torch.bfloat16)
        ops.adapter_dense(given["x"], *args, residual=given["residual"], out=held[:, 8:48])
        assert torch.equal(held[:, 8:48], want) and not held[:, :8].any() and not held[:, 48:].any()
        r = given["residual"].clone()
        ops.adapter_dense(given["x"], *args, residual=r, out=r)
        assert torch.equal(r, want)
    square = layer(40, 40, 40, 1, 40, residual=False)
    for k in ("x", "w"):
        with pytest.raises(ValueError, match="overlap"):
            ops.adapter_dense(square["x"], square["w"], None, square["down"], square["up"], out=square[k])
    for k in ("down", "up"):
        with pytest.raises(ValueError, match="overlap"):
            ops.adapter_dense(square["x"], square["w"], None, square["down"], square["up"], out=square[k][0])


def test_empty_and_refused():
    g = layer(12, 16, 24, 3, 4, index=requests(3, 12), residual=False)
    call = lambda **k: ops.adapter_dense(**({"x": g["x"], "weight": g["w"], "bias": None, "down": g["down"], "up": g["up"], "index": g["index"]} | k))  # noqa: E731
    y, saved = ops.adapter_dense(g["x"][:0], g["w"], None, g["down"], g["up"], g["index"][:0], want_saved=True)
    grads = ops.adapter_dense_backward(y, g["x"][:0], g["w"], None, g["down"], g["up"], g["index"][:0], saved=saved, want_dweight=True)
    assert y.shape == (0, 24) and grads[0].shape == (0, 16) and not any(t.any() for t in (grads[1], grads[3], grads[4]))
    assert torch.equal(call(index=g["index"].long()), call())
    assert torch.equal(call(scale=torch.full((3,), 2.0, device=DEV)), call(scale=2.0))
    assert torch.equal(call(x=g["x"].view(3, 4, 16), index=g["index"][:3]).view(12, 24), call(index=g["index"][:3].repeat_interleave(4)))
    one = torch.tensor(2, device=DEV)
    assert torch.equal(call(index=one), call(index=one.expand(12)))  # an index of no axes is of all rows
    for bad, word in (({"down": g["down"][..., :8]}, "down"), ({"down": g["down"][0]}, "down"), ({"down": g["down"].half()}, "dtype"),
                      ({"up": g["up"][:2]}, "up"), ({"up": g["up"][:, :20]}, "up"), ({"up": g["up"].float()}, "dtype"), ({"index": None}, "index"),
                      ({"index": g["index"][:5]}, "index"), ({"index": g["index"].float()}, "int32"), ({"index": g["index"].cpu()}, "device"),
                      ({"index": g["index"].view(12, 1).expand(12, 16)}, "index"), ({"scale": torch.ones(2, device=DEV)}, "scale"),
                      ({"scale": torch.ones(3, device=DEV, dtype=torch.half)}, "scale"), ({"activation": "swish"}, "activation"),
                      ({"x": g["x"].float(), "weight": g["w"].float()}, "bfloat16"), ({"residual": g["x"]}, "residual")):
        with pytest.raises(ValueError, match=word):
            call(**bad)
    wide = layer(12, 16, 24, 1, 257, residual=False)
    with pytest.raises(ValueError, match="rank"):
        ops.adapter_dense(wide["x"], wide["w"], None, wide["down"], wide["up"])
    y, saved = call(want_saved=True)
    for kept in ((saved[0][:5], None), (saved[0].half(), None), (saved[0], torch.zeros(12, 8, device=DEV)), (None, None)):
        with pytest.raises(ValueError, match="saved"):
            ops.adapter_dense_backward(y, g["x"], g["w"], None, g["down"], g["up"], g["index"], saved=kept)


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
def test_gradients_one_by_one(gated):
    """Each gradient with and without the others."""
    for n, each in ((5, 1), (9, 50), (3, 1600)):
        given = layer(n * each, 72, 96, 4, 12, gated=gated, residual=False, index=requests(4, n))
        x, dy = given["x"].view(n, each, -1), given["dy"].view(n, each, -1)
        args = (given["w"], given["bias"], given["down"], given["up"], given["index"], given["scale"])
        forward, back = (ops.adapter_gated_dense, ops.adapter_gated_dense_backward) if gated else (ops.adapter_dense, ops.adapter_dense_backward)
        _, saved = forward(x, *args, activation="silu", want_saved=True)
        names = ("want_dx", "want_dweight", "want_dbias", "want_ddown", "want_dup")
        full = back(dy, x, *args, activation="silu", saved=saved, **dict.fromkeys(names, True))
        for k, name in enumerate(names):
            got = back(dy, x, *args, activation="silu", saved=saved, **(dict.fromkeys(names, False) | {name: True}))
            for i, t in enumerate(got):
                if i != k:
                    assert t is None
                else:  # (a join in another order, at most)
                    assert (t.double() - full[k].double()).norm() <= 2.0 ** -8 * full[k].double().norm()


def test_gradient_against_differences():
    """Central differences of the formula in 64 bits along random directions of x, D and U."""
    given = layer(90, 40, 48, 3, 8, torch.float16, True, False, False, requests(3, 30, seed=4))
    index = given["index"].long().repeat_interleave(3)

    def f(x, down, up):
        z = x @ given["w"].double().t()
        for g in range(3):
            r = (index == g).nonzero().view(-1)
            z = z.index_add(0, r, float(given["scale"][g]) * x[r] @ down[g].t() @ up[g].t())
        return (z[:, :48] * ACTS["silu"](z[:, 48:]) * given["dy"].double()).sum()

    point = [given[k].double() for k in ("x", "down", "up")]
    args = (given["w"], None, given["down"], given["up"], given["index"], given["scale"])
    y, saved = ops.adapter_gated_dense(given["x"].view(30, 3, -1), *args, want_saved=True)
    dx, _, _, ddown, dup = ops.adapter_gated_dense_backward(given["dy"].view(30, 3, -1), given["x"].view(30, 3, -1), *args, saved=saved)
    for k, have in enumerate((dx.view(90, -1), ddown, dup)):
        for seed in range(3):
            t = randn(*point[k].shape, seed=20 + seed, dtype=torch.float64)
            ends = [f(*(p + s * 1e-5 * t if i == k else p for i, p in enumerate(point))) for s in (1, -1)]
            # each gradient is off by a few roundings of 2^-11
            assert abs((have.double() * t).sum() - (ends[0] - ends[1]) / 2e-5) <= 8 * 2.0 ** -11 * (have.double() * t).norm()


def test_captured_with_another_index_at_each_replay():
    for n, each in ((4, 1), (48, 1), (4, 300)):
        given = layer(n * each, 64, 40, 3, 16, residual=False, bias=False, index=requests(3, n))
        index = given["index"].clone()
        x, dy = given["x"].view(n, each, -1), given["dy"].view(n, each, -1)

        def step():
            y, saved = ops.adapter_dense(x, given["w"], None, given["down"], given["up"], index, given["scale"], activation="relu", want_saved=True)
            return [y, *ops.adapter_dense_backward(dy, x, given["w"], None, given["down"], given["up"], index, given["scale"], activation="relu", saved=saved)]

        step()
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):  # two graphs at once, of one pool
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
                out = step()
            graphs.append((graph, out))
        for seed in range(3):
            index.copy_(requests(3, n, seed=seed))
            want = step()
            for graph, out in graphs:
                graph.replay()
                assert all(a is None or torch.equal(a, b) for a, b in zip(out, want, strict=True))


def test_two_streams_at_once():
    given = [layer(3000, 128, 256, 4, 16, gated=True, residual=False, index=requests(4, 10, seed=s), seed=50 * s) for s in range(2)]

    def step(g):
        args = (g["w"], g["bias"], g["down"], g["up"], g["index"], g["scale"])
        x, dy = g["x"].view(10, 300, -1), g["dy"].view(10, 300, -1)
        y, saved = ops.adapter_gated_dense(x, *args, want_saved=True)
        return [y, *ops.adapter_gated_dense_backward(dy, x, *args, saved=saved)]

    want = [step(g) for g in given]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in given]
    got = []
    for _ in range(5):
        for g, s in zip(given, streams, strict=True):
            with torch.cuda.stream(s):
                got.append(step(g))
    torch.cuda.synchronize()
    for k, one in enumerate(got):
        assert all(a is None or torch.equal(a, b) for a, b in zip(one, want[k % 2], strict=True))


def test_functions_give_the_gradients_of_the_operators():
    for gated in (False, True):
        given = layer(200, 64, 48, 3, 12, gated=gated, index=requests(3, 20))
        x, res, dy = (None if given[k] is None else given[k].view(20, 10, -1) for k in ("x", "residual", "dy"))
        names = ("w", "bias", "down", "up")
        leaves = [x.clone().requires_grad_(True)] + [given[k].clone().requires_grad_(True) for k in names] + ([] if gated else [res.clone().requires_grad_(True)])
        lx, lw, lb, ld, lu, *lr = leaves
        args = (given["w"], given["bias"], given["down"], given["up"], given["index"], given["scale"])
        if gated:
            y = b200.adapter_gated_dense(lx, lw, lb, ld, lu, given["index"], given["scale"])
            want, saved = ops.adapter_gated_dense(x, *args, want_saved=True)
            grads = ops.adapter_gated_dense_backward(dy, x, *args, saved=saved, want_dweight=True, want_dbias=True)
        else:
            y = b200.adapter_dense(lx, lw, lb, ld, lu, given["index"], given["scale"], activation="gelu", residual=lr[0])
            want, saved = ops.adapter_dense(x, *args, activation="gelu", residual=res, want_saved=True)
            grads = (*ops.adapter_dense_backward(dy, x, *args, activation="gelu", saved=saved, want_dweight=True, want_dbias=True), dy)
        assert torch.equal(y, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), grads, strict=True))
    given = layer(30, 16, 24, 1, 4, residual=False, bias=False)
    up = given["up"].clone().requires_grad_(True)
    y = b200.adapter_dense(given["x"], given["w"], None, given["down"], up, scale=0.5)  # only what needs a gradient gets one
    y.sum().backward()
    assert up.grad is not None
    with torch.no_grad():
        assert not b200.adapter_dense(given["x"], given["w"], None, given["down"], up).requires_grad
    with pytest.raises(NotImplementedError, match="scale"):
        b200.adapter_dense(given["x"], given["w"], None, given["down"], up, None, torch.ones(1, device=DEV, requires_grad=True))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        b200.adapter_dense(given["x"], given["w"], None, torch.autograd.forward_ad.make_dual(given["down"], given["down"]), given["up"])
