"""Layer norm, dense and gated dense layers and their gradients, against the formulas in 64 bits.

Tolerances are bounds, derived from the roundings that the operators make: with u half the spacing of the type, a result is
within u * |result| of the formula (one rounding at the end), plus 2^-18 of the sum of the absolute terms for sums in 32 bits
(up to a few thousand terms), plus, behind a gradient before the activation that is rounded between two kernels, u times its
absolute terms.  Slopes are at most 1.2 (the first) and 0.8 (the second derivative of every activation here).
"""

import math

import pytest
import torch

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


def half_spacing(dtype):
    return torch.finfo(dtype).eps / 2


def randn(*shape, seed, dtype=torch.bfloat16, std=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def within(got, want, bound, what):
    excess = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = excess.max().item() if excess.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} over its bound (at most {bound.max().item():.3g})"


# ------------------------------------------------------------------------------------------------------ layer norm


def norm_formula(x, w, b, eps, dy=None):
    x = x.double()
    w = torch.ones_like(x[0]) if w is None else w.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + (0 if b is None else b.double())
    if dy is None:
        return y, xh, rstd
    dy = dy.double()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, xh, rstd, dx, (dy * xh).sum(0), dy.sum(0), g


def check_norm(x, w, b, dy, eps=1e-5):
    """Forward and backward of two-dimensional x against the formula."""
    y, stats = ops.layer_norm(x, w, b, eps, want_stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, stats, w)
    want_y, xh, rstd, want_dx, want_dw, want_db, g = norm_formula(x, w, b, eps, dy)
    u, pu = half_spacing(x.dtype), half_spacing(x.dtype if w is None else w.dtype)
    wa = 1.0 if w is None else w.double().abs()
    # the mean is off by 2^-24 of the largest terms, which rstd carries into every centred value
    shift = SUM * (rstd * x.double().abs().amax(-1, keepdim=True) + xh.abs().amax(-1, keepdim=True))
    within(y, want_y, 1.01 * u * want_y.abs() + shift * wa + 1e-30, "y")
    ga = g.abs().mean(-1, keepdim=True)
    terms = rstd * (g.abs() + ga + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    spread = rstd * shift * ((g * xh).abs().mean(-1, keepdim=True) + xh.abs() * ga + ga)
    within(dx, want_dx, 1.01 * u * want_dx.abs() + SUM * terms + 2 * spread + 1e-30, "dx")
    within(dw, want_dw, 1.01 * pu * want_dw.abs() + SUM * (dy.double() * xh).abs().sum(0) + (dy.double().abs() * shift).sum(0) + 1e-30, "dweight")
    within(db, want_db, 1.01 * pu * want_db.abs() + SUM * dy.double().abs().sum(0) + 1e-30, "dbias")


NORM_SHAPES = [(1, 1), (1, 384), (2, 3), (3, 16), (7, 100), (5, 128), (300, 128), (21, 40), (30, 200), (30, 203), (65, 257), (33, 384), (17, 1001), (40, 1024),
               (9, 2000), (6, 4100), (5, 8192), (3, 12288), (2, 16384), (2, 16383), (5000, 64), (1, 16384)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_layer_norm(rows, width, dtype):
    x, dy = randn(rows, width, seed=1, dtype=dtype, std=1.5, mean=0.25), randn(rows, width, seed=2, dtype=dtype, std=0.1)
    kind = torch.float32 if (rows + width) % 2 else dtype
    w, b = randn(width, seed=3, dtype=kind, std=0.2, mean=1.0), randn(width, seed=4, dtype=kind)
    check_norm(x, w, b, dy)


def test_layer_norm_of_many_rows():
    x, dy = randn(70001, 128, seed=1, std=1.5, mean=0.25), randn(70001, 128, seed=2, std=0.1)
    w, b = randn(128, seed=3, dtype=torch.float32, mean=1.0), randn(128, seed=4, dtype=torch.float32)
    check_norm(x, w, b, dy)


def test_layer_norm_without_parameters_and_with_a_weight_alone():
    x, dy = randn(37, 200, seed=1), randn(37, 200, seed=2)
    check_norm(x, None, None, dy)
    check_norm(x, randn(200, seed=3), None, dy)


def test_layer_norm_of_rows_with_a_large_mean_and_of_constant_rows():
    x = randn(9, 512, seed=1, dtype=torch.float32, mean=1000.0)
    check_norm(x, None, None, randn(9, 512, seed=2, dtype=torch.float32))
    flat = torch.full((4, 96), 3.5, device=DEV, dtype=torch.bfloat16)
    y, stats = ops.layer_norm(flat, None, None, 1e-5, want_stats=True)
    assert (y == 0).all() and torch.allclose(stats[:, 0], torch.full((4,), 1e-5 ** -0.5, device=DEV), rtol=1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(3000, 1), (2500, 5), (2500, 9), (3001, 15), (2000, 24), (1500, 127), (700, 519), (900, 4093), (310, 8190)])
def test_layer_norm_rows_on_other_boundaries(rows, width, dtype):
    """Rows of odd pitches and offsets, more of them than run at once: x, dy and the results each on boundaries of their own."""
    wide = width + 6
    x, dy = (randn(rows * wide + 16, seed=s, dtype=dtype, std=d) for s, d in ((1, 1.5), (2, 0.1)))
    w, b = randn(width + 1, seed=3, dtype=dtype, mean=1.0)[1:], randn(width + 1, seed=4, dtype=dtype)[1:]
    for x_first, x_pitch, dy_first, dy_pitch in ((0, width, 0, width), (3, width + 1, 1, width), (5, width + 2, 2, width + 5)):
        xs = x[x_first:].as_strided((rows, width), (x_pitch, 1))
        dys = dy[dy_first:].as_strided((rows, width), (dy_pitch, 1))
        check_norm(xs, w, b, dys)
        held, again = (torch.zeros(rows * wide + 8, device=DEV, dtype=dtype) for _ in range(2))
        places = [t[1:].as_strided((rows, width), (wide - 1, 1)) for t in (held, again)]
        ops.layer_norm(xs, w, b, out=places[0])
        ops.layer_norm(xs.contiguous(), w, b, out=places[1])  # the same rows to the same boundaries: the same sums
        assert torch.equal(held, again)
        places[0].zero_()
        assert not held.any()


@pytest.mark.parametrize("rows,width", [(1, 300), (4, 317), (40, 384), (60, 200), (2000, 8), (1237, 1001), (500, 8192)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_gradients_one_by_one(rows, width, dtype):
    """Each of dx, dweight and dbias with and without the others, and nothing written behind the workspace."""
    x, dy, w = (randn(*shape, seed=i, dtype=dtype) for i, shape in enumerate(((rows, width), (rows, width), (width,))))
    stats = ops.layer_norm(x, w, want_stats=True)[1]
    code = _lib.DTYPE_BF16 if dtype == torch.bfloat16 else _lib.DTYPE_F32
    need = _lib.load().b200ta_layer_norm_workspace_bytes(rows, width)
    held = torch.empty(need + (1 << 20), device=DEV, dtype=torch.uint8)
    wanted = {}
    for want in [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)]:
        held.fill_(0x5A)
        out = {"dx": torch.zeros_like(x), "dweight": torch.zeros_like(w), "dbias": torch.zeros_like(w)}
        dx, dw, db = (t.data_ptr() if on else None for t, on in zip(out.values(), want, strict=True))
        _lib.call("b200ta_layer_norm_backward", dy.data_ptr(), width, x.data_ptr(), width, stats.data_ptr(), w.data_ptr(), code, dx, width, dw, db,
                  held.data_ptr(), need, code, rows, width, torch.cuda.current_stream().cuda_stream)
        assert (held[need:] == 0x5A).all(), want
        for (name, t), on in zip(out.items(), want, strict=True):
            assert torch.equal(t, wanted.setdefault(name, t)) if on else not t.any(), (name, want)


def test_layer_norm_strides_and_leading_shapes():
    base = randn(6, 5, 3, 160, seed=1)
    for x in (base[..., 7:107], base[:, 1:4, :, ::2], base.transpose(0, 2), base[:, :, 1], base.permute(0, 1, 3, 2), base[:0],
              base[..., :1].expand(6, 5, 3, 40), base[:1].expand(4, 5, 3, 160)):
        width = x.shape[-1]
        w, dy = randn(width, seed=3, mean=1.0), randn(*x.shape, seed=2)
        y, stats = ops.layer_norm(x, w, None, 1e-5, want_stats=True)
        want, want_stats = ops.layer_norm(x.contiguous(), w, None, 1e-5, want_stats=True)
        assert torch.equal(y, want) and torch.equal(stats, want_stats) and y.shape == x.shape
        got = ops.layer_norm_backward(dy, x, stats, w)
        for a, b in zip(got, ops.layer_norm_backward(dy.clone(), x.contiguous(), stats, w), strict=True):
            assert torch.equal(a, b)
    out = torch.zeros(6, 200, device=DEV, dtype=torch.bfloat16)
    x = randn(6, 160, seed=5)
    ops.layer_norm(x, out=out[:, 8:168])
    assert torch.equal(out[:, 8:168], ops.layer_norm(x)) and (out[:, :8] == 0).all() and (out[:, 168:] == 0).all()


def test_layer_norm_keeps_infinities_and_nan_in_their_rows():
    x, dy = randn(64, 128, seed=1), randn(64, 128, seed=2)
    bad = x.clone()
    bad[3, 5], bad[40, 0] = math.nan, math.inf
    y, stats = ops.layer_norm(bad, want_stats=True)
    dx = ops.layer_norm_backward(dy, bad, stats)[0]
    clean_y, clean_stats = ops.layer_norm(x, want_stats=True)
    clean_dx = ops.layer_norm_backward(dy, x, clean_stats)[0]
    rest = torch.ones(64, dtype=torch.bool, device=DEV)
    rest[[3, 40]] = False
    assert torch.equal(y[rest], clean_y[rest]) and torch.equal(dx[rest], clean_dx[rest])
    assert y[~rest].isnan().all() and dx[~rest].isnan().all()


def test_layer_norm_gradient_against_differences():
    """Central differences of the formula in 64 bits along random directions."""
    x, dy, w = (randn(*s, seed=i, dtype=torch.float32) for i, s in enumerate([(11, 130), (11, 130), (130,)]))
    _, stats = ops.layer_norm(x, w, None, 1e-5, want_stats=True)
    dx, dw, _ = ops.layer_norm_backward(dy, x, stats, w)
    h = 1e-5
    for seed in range(3):
        t = randn(11, 130, seed=10 + seed, dtype=torch.float64)
        f = [(norm_formula(x.double() + s * h * t, w, None, 1e-5)[0] * dy).sum() for s in (1, -1)]
        assert abs((dx.double() * t).sum() - (f[0] - f[1]) / (2 * h)) < 1e-4 * (dx.double() * t).abs().sum()
        t = randn(130, seed=20 + seed, dtype=torch.float64)
        f = [(norm_formula(x, w.double() + s * h * t, None, 1e-5)[0] * dy).sum() for s in (1, -1)]
        assert abs((dw.double() * t).sum() - (f[0] - f[1]) / (2 * h)) < 1e-4 * (dw.double() * t).abs().sum()


# ---------------------------------------------------------------------------------------------- dense, gated dense


def layer_formula(x, w, bias, residual, activation, gated, dy=None):
    """y and the terms of its sums; with dy also (dz, dx, dweight, dbias), by the formulas in 64 bits."""
    x, w = x.double(), w.double()
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    act = ACTS[activation]
    t = (z[:, z.shape[1] // 2:] if gated else z).clone().requires_grad_(True)
    with torch.enable_grad():
        a = act(t)
        slope = torch.autograd.grad(a.sum(), t)[0]
    a = a.detach()
    if gated:
        n = z.shape[1] // 2
        value, gate = z[:, :n], z[:, n:]
        y, terms = value * a, size[:, :n] * a.abs() + value.abs() * 1.2 * size[:, n:]
    else:
        y, terms = a, 1.2 * size
        if residual is not None:
            y, terms = y + residual.double(), terms + residual.double().abs()
    if dy is None:
        return y, terms
    dy = dy.double()
    if gated:
        dz = torch.cat([dy * a, dy * value * slope], 1)
        sums = torch.cat([1.2 * dy.abs() * size[:, n:], dy.abs() * (size[:, :n] * 1.2 + 0.8 * value.abs() * size[:, n:])], 1)
    else:
        dz = dy * slope
        sums = 0.8 * dy.abs() * size
    return y, terms, dz, sums


def check_layer(x, w, bias=None, residual=None, activation="none", gated=False, dy=None, keep=None):
    """Forward, and with dy backward (with what the forward pass keeps, or without), of two-dimensional x."""
    u = half_spacing(x.dtype)
    tiny = torch.finfo(x.dtype).smallest_normal
    if gated:
        got, saved = ops.gated_dense(x, w, bias, activation=activation, want_saved=True)
    else:
        got, saved = ops.dense(x, w, bias, activation=activation, residual=residual, want_saved=True)
    y, terms = layer_formula(x, w, bias, residual, activation, gated)
    within(got, y, 1.01 * u * y.abs() + SUM * terms + tiny, "y")
    if dy is None:
        return
    if keep is False:
        saved = None
    back = ops.gated_dense_backward if gated else ops.dense_backward
    dx, dw, db = back(dy, x, w, bias, activation=activation, saved=saved, want_dbias=True)
    _, _, dz, sums = layer_formula(x, w, bias, residual, activation, gated, dy)
    # dz is rounded where a kernel hands it to the next one
    plain = activation == "none" and not gated
    off = SUM * sums + (0 if plain else 1.01 * u * dz.abs() + tiny)
    if activation == "relu":  # its slope jumps: where a sum in 32 bits may have the other sign, either is right
        z = x.double() @ w.double().t() + (0 if bias is None else bias.double())
        g = z[:, z.shape[1] // 2:] if gated else z
        near = g.abs() < SUM * (x.double().abs() @ w.double().abs().t() + 1)[:, -g.shape[1]:]
        jump = near * dy.double().abs() * (z[:, :g.shape[1]].abs() if gated else 1)
        off = off + (torch.cat([torch.zeros_like(jump), jump], 1) if gated else jump)
    xd, wd = x.double(), w.double()
    for name, have, want, bound in (("dx", dx, dz @ wd, off @ wd.abs() + SUM * (dz.abs() @ wd.abs())),
                                    ("dweight", dw, dz.t() @ xd, off.t() @ xd.abs() + SUM * (dz.abs().t() @ xd.abs())),
                                    ("dbias", db, dz.sum(0), off.sum(0) + SUM * dz.abs().sum(0))):
        within(have, want, 1.01 * u * want.abs() + bound + tiny, name)


def layer_inputs(rows, K, N, dtype, gated, bias, residual, seed=0):
    columns = 2 * N if gated else N
    return {
        "x": randn(rows, K, seed=seed + 1, dtype=dtype),
        "w": randn(columns, K, seed=seed + 2, dtype=dtype, std=K ** -0.5),
        "bias": randn(columns, seed=seed + 3, dtype=dtype, std=0.3) if bias else None,
        "residual": randn(rows, N, seed=seed + 4, dtype=dtype) if residual and not gated else None,
        "gated": gated,
        "dy": randn(rows, N, seed=seed + 5, dtype=dtype, std=0.1),
    }


# rows around the few-rows limit and the tiles of 128, widths around 8, 32, 64 and the tiles of 64, 128 and 256
SIZES = [(1, 1, 1), (1, 384, 96), (2, 8, 8), (3, 15, 7), (5, 64, 33), (16, 100, 130), (17, 64, 64), (31, 40, 24), (100, 16, 16),
         (128, 128, 128), (129, 72, 65), (200, 515, 129), (257, 128, 512), (300, 384, 200), (500, 1, 40), (333, 1000, 1),
         (1000, 96, 320), (2500, 520, 136), (700, 1030, 133), (200, 1541, 70)]


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_layer_sizes(rows, K, N, gated):
    more = (rows + K + N) % 2 == 0
    dtype = torch.float16 if (rows + N) % 3 == 0 else torch.bfloat16
    check_layer(activation="silu", **layer_inputs(rows, K, N, dtype, gated, more, not more))


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("activation", list(ACTS))
@pytest.mark.parametrize("rows,K", [(6, 64), (150, 64), (150, 1544)])
def test_layer_activations(rows, K, activation, gated):
    """Few rows, pre-activations computed again, pre-activations kept."""
    for dtype in (torch.bfloat16, torch.float16):
        check_layer(activation=activation, **layer_inputs(rows, K, 72, dtype, gated, True, True))


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
def test_kept_and_computed_pre_activations(gated):
    given = layer_inputs(400, 1600, 264, torch.bfloat16, gated, True, True)
    check_layer(activation="gelu", **given)
    check_layer(activation="gelu", keep=False, **given)


@pytest.mark.parametrize("rows,K,N,gated", [(150000, 128, 512, True), (270001, 16, 1024, True), (300001, 24, 1000, False)])
def test_rows_in_chunks(rows, K, N, gated):
    """The last two have so many rows that the backward pass takes them in several chunks."""
    check_layer(activation="silu", **layer_inputs(rows, K, N, torch.bfloat16, gated, True, False))


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows,K,N", [(9472, 128, 64), (9700, 64, 200), (10001, 128, 512), (12000, 8, 7), (9999, 72, 130)])
def test_narrow_layers_of_many_rows(rows, K, N, gated):
    """At most 128 inputs: dz and dx come from one kernel.  Rows and units that fill its tiles of 256 and 64, and do not."""
    dtype = torch.float16 if N % 4 else torch.bfloat16
    given = layer_inputs(rows, K, N, dtype, gated, rows % 2 == 0, False)
    check_layer(activation="silu", **given)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    back = ops.gated_dense_backward if gated else ops.dense_backward
    both, alone = back(dy, x, w, bias, activation="gelu"), back(dy, x, w, bias, activation="gelu", want_dweight=False, want_dbias=False)
    assert torch.equal(both[0], alone[0]) and alone[1] is None


def test_sums_of_many_parts_of_narrow_tiles():
    """db from dW's product with few inputs: several tiles a block, with their sums beside them."""
    check_layer(activation="relu", **layer_inputs(136787, 24, 160, torch.bfloat16, True, True, False))


@pytest.mark.parametrize("rows,K,N,gated", [(9600, 104, 1000, True), (3000, 64, 640, False), (1000, 40, 3000, True), (2047, 520, 1288, False), (300, 1600, 264, True)])
def test_the_workspace_is_enough_for_every_choice_of_gradients(rows, K, N, gated):
    """Each of dx, dW and db with and without the others: nothing is written behind the workspace, and what is wanted is the same."""
    given = layer_inputs(rows, K, N, torch.bfloat16, gated, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    gelu, bf16, outer = 3, 0, 2 if gated else 1
    needs = [_lib.load().b200ta_dense_backward_workspace_bytes(gelu, gated, 0, want_dbias, rows, K, N) for want_dbias in (0, 1)]
    held = torch.empty(max(needs) + (64 << 20), device=DEV, dtype=torch.uint8)
    wanted = {}
    for want in [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)]:
        held.fill_(0x5A)
        need = needs[want[2]]
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(outer * N, device=DEV, dtype=x.dtype)
        dx_p, dw_p, db_p = (t.data_ptr() if on else None for t, on in zip((dx, dw, db), want, strict=True))
        _lib.call("b200ta_dense_backward", dy.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, bias.data_ptr(), None, 0, dx_p, K, dw_p, db_p,
                  held.data_ptr(), need, bf16, gelu, gated, rows, K, N, torch.cuda.current_stream().cuda_stream)
        assert (held[need:] == 0x5A).all(), want
        for name, t, on in zip(("dx", "dw", "db"), (dx, dw, db), want, strict=True):
            if not on:
                assert not t.any()
            elif name == "dx":
                assert torch.equal(t, wanted.setdefault(name, t)), want
            else:  # their sums may run in another order: one rounding apart, and 32-bit sums of rows values of 1 or so
                first = wanted.setdefault(name, t.double())
                within(t, first, 2.02 * half_spacing(t.dtype) * first.abs() + 4 * SUM * rows, name)


def test_parts_of_the_weight_gradient():
    """dW in one piece, and in parts of the rows."""
    check_layer(**layer_inputs(256, 2048, 2048, torch.bfloat16, False, True, True))
    check_layer(**layer_inputs(20000, 64, 64, torch.bfloat16, False, True, True))


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows,K,N", [(40, 33, 6000), (300, 130, 5001), (129, 1024, 4096)])
def test_parts_of_the_input_gradient(rows, K, N, gated):
    """Few rows and many hidden units: dx in parts of the units, with and without the other gradients beside it."""
    given = layer_inputs(rows, K, N, torch.bfloat16, gated, True, False)
    check_layer(activation="silu", **given)
    back = ops.gated_dense_backward if gated else ops.dense_backward
    both = back(given["dy"], given["x"], given["w"], given["bias"], activation="silu")
    alone = back(given["dy"], given["x"], given["w"], given["bias"], activation="silu", want_dweight=False, want_dbias=False)
    assert torch.equal(both[0], alone[0]) and alone[1] is None


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows,K,N", [(1, 8, 16), (2, 33, 17), (7, 1703, 130), (8, 520, 15), (9, 100, 300), (13, 31, 257), (16, 1030, 64), (16, 4096, 40)])
def test_few_rows(rows, K, N, gated):
    """Up to 16 rows: one and two groups of eight, columns and inputs that fill the products and do not."""
    for dtype in (torch.bfloat16, torch.float16):
        check_layer(activation="gelu", **layer_inputs(rows, K, N, dtype, gated, True, not gated))


def test_activations_far_out():
    """Slopes and values where exponentials overflow, and NaN, pass column by column."""
    z = torch.tensor([0.0, -0.0, 1e-3, -5, 5, -20, 20, -44, 44, -90, 90, -1e4, 1e4, -1e15, 1e15, -3e38, 3e38], device=DEV)
    for rows in (1, 40):
        x = torch.ones(rows, 8, device=DEV, dtype=torch.bfloat16)
        w = torch.zeros(z.numel(), 8, device=DEV, dtype=torch.bfloat16)
        w[:, 0] = z
        zr = w[:, 0].double()
        for name, act in ACTS.items():
            y = ops.dense(x, w, activation=name)
            want = act(zr)
            want = torch.where(want.isnan(), zr.clamp(min=0) if name != "sigmoid" else (zr > 0).double(), want)
            torch.testing.assert_close(y[-1].double(), want, rtol=2 ** -7, atol=1e-6)
            ones = torch.ones(rows, z.numel(), device=DEV, dtype=torch.bfloat16)
            db = ops.dense_backward(ones, x, w, activation=name, want_dbias=True)[2]
            assert torch.isfinite(db).all(), name
            slope = db.double() / rows
            far = zr.abs() >= 44
            limit = torch.where(zr > 0, 1.0, 0.0).double() if name not in ("none", "sigmoid") else torch.full_like(zr, float(name == "none"))
            torch.testing.assert_close(slope[far], limit[far], rtol=2 ** -6, atol=1e-6)
        w[3, 1] = math.nan
        for name in ACTS:
            y = ops.dense(x, w, activation=name)
            assert y[:, 3].isnan().all() and not y[:, [2, 4]].isnan().any(), name


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows", [5, 90])
def test_strides_and_alignment(rows, gated):
    """Views of every kind give what their contiguous copies give."""
    K, N = 48, 40
    columns = 2 * N if gated else N
    fwd = ops.gated_dense if gated else ops.dense
    back = ops.gated_dense_backward if gated else ops.dense_backward
    wide, tall = randn(rows, 2 * K + 16, seed=1), randn(K, rows + 3, seed=2)
    xs = [wide[:, :K], wide[:, 3:3 + K], wide[:, ::2][:, :K], tall.t()[:rows], wide[:1, :K].expand(rows, K),
          randn(2, rows, K, seed=3)[1], randn(rows * K + 1, seed=4)[1:].view(rows, K)]
    big = randn(columns, 2 * K, seed=5, std=K ** -0.5)
    ws = [big[:, :K], big[:, 1:1 + K], big[:, ::2], randn(K, columns, seed=6, std=K ** -0.5).t(), big[:, :K].contiguous()]
    dys = [randn(rows, N, seed=7), randn(N, rows, seed=8).t(), randn(rows, 1, seed=9).expand(rows, N), randn(1, 1, seed=9).expand(rows, N),
           randn(rows, N + 5, seed=10)[:, 5:]]
    bias = randn(columns + 1, seed=11)[1:]
    for i in range(max(len(xs), len(ws), len(dys))):
        x, w, dy = xs[i % len(xs)], ws[i % len(ws)], dys[i % len(dys)]
        y = fwd(x, w, bias, activation="silu")
        assert torch.equal(y, fwd(x.contiguous(), w.contiguous(), bias.clone(), activation="silu")), i
        got = back(dy, x, w, bias, activation="silu")
        want = back(dy.contiguous(), x.contiguous(), w.contiguous(), bias.clone(), activation="silu")
        for a, b in zip(got, want, strict=True):
            assert torch.equal(a, b), i
        for where in (torch.zeros(rows, N + 16, device=DEV, dtype=torch.bfloat16)[:, 8:8 + N],
                      torch.zeros(rows, N + 9, device=DEV, dtype=torch.bfloat16)[:, 3:3 + N]):
            fwd(x, w, bias, activation="silu", out=where)
            assert torch.equal(where, y)
            whole = torch.as_strided(where, (rows, where.stride(0)), (where.stride(0), 1), 0)
            assert (whole[:, :where.storage_offset()] == 0).all() and (whole[:, where.storage_offset() + N:] == 0).all()


def test_leading_shapes():
    x = randn(2, 3, 50, 64, seed=1)
    w = randn(80, 64, seed=2, std=0.1)
    res = randn(2, 50, 3, 80, seed=3).transpose(1, 2)
    y = ops.dense(x, w, residual=res)
    assert torch.equal(y, ops.dense(x.view(-1, 64), w, residual=res.reshape(-1, 80)).view(2, 3, 50, 80))
    y = ops.gated_dense(x.transpose(0, 1), w)
    assert y.shape == (3, 2, 50, 40) and torch.equal(y, ops.gated_dense(x, w).transpose(0, 1))
    assert ops.dense(x[:0], w).shape == (0, 3, 50, 80) and ops.gated_dense(x[0, 0, 0], w).shape == (40,)
    dx, dw, db = ops.dense_backward(torch.empty(0, 80, device=DEV, dtype=torch.bfloat16), x.view(-1, 64)[:0], w, want_dbias=True)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_only_what_is_wanted():
    given = layer_inputs(300, 64, 72, torch.bfloat16, True, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    whole = ops.gated_dense_backward(dy, x, w, bias)
    for k in range(3):
        wanted = {n: i == k for i, n in enumerate(("want_dx", "want_dweight", "want_dbias"))}
        got = ops.gated_dense_backward(dy, x, w, bias, **wanted)
        assert [g is None for g in got] == [i != k for i in range(3)] and torch.equal(got[k], whole[k])
    y, stats = ops.layer_norm(x, want_stats=True)
    assert ops.layer_norm_backward(x, x, stats, want_dx=False, want_dweight=False, want_dbias=False) == (None, None, None)


def test_results_repeat_bit_by_bit_and_on_another_stream():
    given = layer_inputs(5000, 96, 200, torch.bfloat16, True, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]

    def everything():
        y, stats = ops.layer_norm(x, want_stats=True)
        h = ops.gated_dense(y, w, bias)
        return [y, h, *ops.gated_dense_backward(dy, y, w, bias), *ops.layer_norm_backward(x, x, stats)]

    first = everything()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = everything()
    side.synchronize()
    third = everything()
    for a, b, c in zip(first, second, third, strict=True):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_calls_in_a_graph():
    given = layer_inputs(700, 96, 200, torch.bfloat16, True, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]

    def step():
        y, saved = ops.gated_dense(x, w, bias, want_saved=True)
        return [y, *ops.gated_dense_backward(dy, x, w, bias, saved=saved)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(randn(700, 96, seed=77))
    graph.replay()
    for a, b in zip(out, step(), strict=True):
        assert torch.equal(a, b)


def test_rows_with_nan_stay_in_their_rows():
    given = layer_inputs(200, 64, 72, torch.bfloat16, True, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    bad = x.clone()
    bad[130, 3] = math.nan
    keep = torch.arange(200, device=DEV) != 130
    y, clean = ops.gated_dense(bad, w, bias), ops.gated_dense(x, w, bias)
    assert torch.equal(y[keep], clean[keep]) and y[130].isnan().all()
    dx = ops.gated_dense_backward(dy, bad, w, bias)[0]
    assert torch.equal(dx[keep], ops.gated_dense_backward(dy, x, w, bias)[0][keep]) and dx[130].isnan().all()


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
def test_gradients_against_differences(gated):
    """Central differences of the formula in 64 bits along random directions; the gradients are rounded to fp16, and dz before
    them: 2^-11 each of the terms they sum."""
    given = layer_inputs(60, 40, 24, torch.float16, gated, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    back = ops.gated_dense_backward if gated else ops.dense_backward
    dx, dw, db = back(dy, x, w, bias, activation="gelu")
    h = 1e-6

    def loss(x, w, bias):
        return (layer_formula(x, w, bias, None, "gelu", gated)[0] * dy.double()).sum()

    args = [x.double(), w.double(), bias.double()]
    dz = layer_formula(x, w, bias, None, "gelu", gated, dy)[2].abs()
    sizes = [dz @ w.double().abs(), dz.t() @ x.double().abs(), dz.sum(0)]
    for k, grad in enumerate((dx, dw, db)):
        for seed in range(2):
            t = randn(*grad.shape, seed=50 + seed, dtype=torch.float64)
            f = [loss(*[a + s * h * t if i == k else a for i, a in enumerate(args)]) for s in (1, -1)]
            tol = 2 * 2.0 ** -11 * (sizes[k] * t.abs()).sum() + 1e-6
            assert abs((grad.double() * t).sum() - (f[0] - f[1]) / (2 * h)) < tol


def test_refusals():
    x, w = randn(20, 32, seed=1), randn(48, 32, seed=2)
    for call in (lambda: ops.dense(x.float(), w.float()), lambda: ops.dense(x, w.half()), lambda: ops.dense(x, w[:, :16]),
                 lambda: ops.dense(x, w, activation="tanh"), lambda: ops.dense(x, w, w[:, 0][:40]), lambda: ops.dense(x, w.cpu()),
                 lambda: ops.dense(x, w, residual=x), lambda: ops.dense(x, w, out=x), lambda: ops.gated_dense(x, w[:47]),
                 lambda: ops.dense(x, w, out=randn(48, 20, seed=3).t()), lambda: ops.dense(x[:, :0], w[:, :0]),
                 lambda: ops.dense_backward(x, x, w), lambda: ops.dense_backward(randn(20, 48, seed=4), x, w, saved=x, activation="silu"),
                 lambda: ops.layer_norm(x, w[0].half()), lambda: ops.layer_norm(x, w[0][:16]), lambda: ops.layer_norm(x, None, w[0]),
                 lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(randn(1, 16385, seed=1)), lambda: ops.layer_norm(x.cpu()),
                 lambda: ops.layer_norm(x, out=w), lambda: ops.layer_norm_backward(x, x, x, None),
                 lambda: ops.layer_norm_backward(w, x, randn(20, 2, seed=1, dtype=torch.float32))):
        with pytest.raises(ValueError):
            call()
