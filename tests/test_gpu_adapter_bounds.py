"""Adapters' gradients within what is rounded, in fp16 and of few rows, and many more adapters than tiles.

The bounds of the adapters' tests add the smallest normal number to each value that is rounded, 2^-14 in fp16, several times a rounding of
gradients around 0.1.  Here gradients are 512 times as large (a power of two: they keep their bits), so that it is below a tenth of the
roundings of most of them."""

import pytest
import torch

from bionemo_inference_runtime_b200 import _lib, ops
from tests.test_gpu_adapters import ACTS, check, layer, requests, within

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    _lib.reset_device_status()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("n,each,K,N,rank", [(6, 1, 64, 72, 16), (50, 1, 64, 72, 12), (30, 5, 200, 72, 20), (3, 300, 136, 96, 16), (3, 300, 520, 40, 40),
                                             (4, 2500, 72, 64, 16)])
def test_fp16_gradients_within_their_roundings(n, each, K, N, rank, activation, gated):
    given = layer(n * each, K, N, 3, rank, torch.float16, gated, True, True, requests(3, n))
    given["dy"] = given["dy"] * 512
    check(activation=activation, **given)


@pytest.mark.parametrize("rows,count", [(50, 16383), (3000, 5000), (10000, 2000)])
@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
def test_thousands_of_adapters(rows, count, gated):
    """Each row its own adapter, from anywhere among them: relative to the size of each result, in bf16 with at most three roundings on the
    way (2^-9 each in the root mean square).  The last adapter and the one behind it are asked for as well; adapters without rows
    have gradients of zero."""
    K, N, rank = 40, 24, 6
    g = torch.Generator(device=DEV).manual_seed(1)
    index = torch.randint(0, count, (rows,), generator=g, device=DEV)
    index[0], index[1], index[2] = count - 1, count, -1
    p = layer(rows, K, N, count, rank, gated=gated, residual=False, index=index)
    forward, back = (ops.adapter_gated_dense, ops.adapter_gated_dense_backward) if gated else (ops.adapter_dense, ops.adapter_dense_backward)
    args = (p["w"], p["bias"], p["down"], p["up"], index, p["scale"])
    y, saved = forward(p["x"], *args, activation="silu", want_saved=True)
    dx, _, _, ddown, dup = back(p["dy"], p["x"], *args, activation="silu", saved=saved)

    x, w, b, down, up = (p[k].double().requires_grad_(True) for k in ("x", "w", "bias", "down", "up"))
    has = index.clamp(0, count - 1)
    share = (p["scale"].double()[has] * ((index >= 0) & (index < count))).unsqueeze(1)
    t = share * torch.einsum("rk,rjk->rj", x, down[has])
    z = x @ w.t() + b + torch.einsum("rj,rnj->rn", t, up[has])
    want = z[:, :N] * torch.nn.functional.silu(z[:, N:]) if gated else torch.nn.functional.silu(z)
    grads = torch.autograd.grad(want, (x, down, up), p["dy"].double())
    for name, got, ref in zip(("y", "dx", "ddown", "dup"), (y, dx, ddown, dup), (want.detach(), *grads), strict=True):
        assert torch.isfinite(got).all() and ((got.double() - ref).norm() / ref.norm()).item() < 3 * 2 ** -9, name
    idle = torch.ones(count, dtype=torch.bool, device=DEV)
    idle[index[(index >= 0) & (index < count)]] = False
    assert idle.any() and not ddown[idle].any() and not dup[idle].any()


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("n,each,K,N,rank,count", [(1, 1, 16, 46, 12, 3), (2, 1, 25, 2584, 16, 9), (4, 1, 520, 40, 33, 4), (1, 2, 64, 16, 58, 2), (16, 1, 72, 300, 16, 5),
                                                   (2, 8, 136, 65, 8, 2), (4, 4, 1032, 520, 100, 8), (13, 4, 80, 16, 64, 7), (100, 5, 128, 24, 16, 6),
                                                   (1000, 1, 64, 56, 16, 6)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_few_rows_carry_their_own_rounding_alone(n, each, K, N, rank, count, activation, gated, dtype):
    """dx of up to 16 rows and db of up to 1024, from the values before the activation that the forward pass kept: the formula in 64 bits, with u
    half the spacing of the type: the result rounded by u, dz by u^2 (for db not at all) and 2^-16 for its slope in 32 bits, dt by u^2, sums in 32 bits by
    2^-18 of their terms."""
    rows = n * each
    p = layer(rows, K, N, count, rank, dtype, gated, True, False, requests(count, n, seed=3))
    p["dy"] = p["dy"] * 64
    index = p["index"]
    forward, back = (ops.adapter_gated_dense, ops.adapter_gated_dense_backward) if gated else (ops.adapter_dense, ops.adapter_dense_backward)
    args = (p["w"], p["bias"], p["down"], p["up"], index, p["scale"])
    x, dy = p["x"].view(n, each, -1), p["dy"].view(n, each, -1)
    _, saved = forward(x, *args, activation=activation, want_saved=True)
    dx, _, dbias, _, _ = back(dy, x, *args, activation=activation, saved=saved, want_dweight=True, want_dbias=True)

    u, least, slope, total = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal, 2.0 ** -16, 2.0 ** -18
    z = saved[1].double().view(rows, 2 if gated else 1, -1)[..., :N]
    pre = z[:, -1].clone().requires_grad_(True)
    a = ACTS[activation](pre)
    s = torch.autograd.grad(a.sum(), pre)[0]
    a, d = a.detach(), p["dy"].double()
    dz = torch.cat([d * a, d * z[:, 0] * s], 1) if gated else d * s
    size = torch.cat([d.abs() * a.abs(), d.abs() * z[:, 0].abs()], 1) if gated else d.abs()  # what a slope's error is of
    off = slope * size + 1.01 * u * u * dz.abs() + least * u
    wd, has = p["w"].double(), index.long().repeat_interleave(each)
    want, bound = dz @ wd, off @ wd.abs() + total * (dz.abs() @ wd.abs())
    for g in range(count):
        r = (has == g).nonzero().view(-1)
        down, up, scale = p["down"][g].double(), p["up"][g].double(), float(p["scale"][g])
        dt, terms = scale * dz[r] @ up, scale * dz[r].abs() @ up.abs()
        want[r] += dt @ down
        dt_off = scale * off[r] @ up.abs() + total * terms + 1.01 * u * u * dt.abs() + least * u
        bound[r] += dt_off @ down.abs() + total * (dt.abs() @ down.abs())
    if rows <= 16:
        within(dx.view(rows, K), want, 1.01 * u * want.abs() + bound + least, "dx")
    want = dz.sum(0)
    within(dbias, want, 1.01 * u * want.abs() + (slope * size + total * dz.abs()).sum(0) + least, "dbias")
