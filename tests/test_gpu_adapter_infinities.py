"""Infinities in rows, in their gradients and in an adapter's own weights: what the formula makes of them, whatever kernels run."""

import math

import pytest
import torch

from bionemo_inference_runtime_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    _lib.reset_device_status()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def positive(*shape, seed, dtype, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.rand(*shape, generator=g, device=DEV) * std + 0.25 * std).to(dtype)


# (rows, rank): values made in each block, beside the few rows, by warp-wide products and by tiles of the tensor cores, of ranks that
# blocks of 16 and of 32 do not divide
WAYS = [(2, 12), (40, 12), (300, 12), (700, 12), (700, 20), (700, 100), (9000, 12), (9000, 16)]


@pytest.mark.parametrize("rows,rank", WAYS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_infinite_row_is_infinite(rows, rank, dtype):
    """With weights of one sign all sums of a row with an infinity are that infinity, forward and backward."""
    x, dy = positive(rows, 72, seed=1, dtype=dtype), positive(rows, 40, seed=2, dtype=dtype)
    layers = (positive(40, 72, seed=3, dtype=dtype, std=0.1), None, positive(1, rank, 72, seed=4, dtype=dtype, std=0.1),
              positive(1, 40, rank, seed=5, dtype=dtype, std=0.1))

    def run(x, dy):
        y, saved = ops.adapter_dense(x, *layers, want_saved=True)
        return y, ops.adapter_dense_backward(dy, x, *layers, saved=saved)[0]

    clean = run(x, dy)
    bad_x, bad_dy = x.clone(), dy.clone()
    row = rows * 2 // 3
    bad_x[row, 5], bad_dy[row, 7] = math.inf, math.inf
    for got, want in zip((run(bad_x, dy)[0], run(x, bad_dy)[1]), clean, strict=True):
        assert (got[row] == math.inf).all()
        others = torch.arange(rows, device=DEV) != row
        assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("n,each", [(6, 1), (48, 1), (200, 1), (12, 40), (6, 256), (40, 100), (4, 3000)])
@pytest.mark.parametrize("rank", [12, 20])
def test_infinite_weights_of_an_adapter_in_its_own_rows(n, each, rank):
    """They make the results infinite or NaN where they make those of the formula so, and nowhere else."""
    g = torch.Generator(device=DEV).manual_seed(3)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV).bfloat16()  # noqa: E731
    x, w, down, up, dy = randn(n, each, 72), randn(40, 72), randn(4, rank, 72), randn(4, 40, rank), randn(n, each, 40)
    index = torch.arange(n, device=DEV, dtype=torch.int32) % 5  # (4 is none)
    up[1, 7, 2], down[2, 3, 5] = math.inf, -math.inf
    y, saved = ops.adapter_dense(x, w, None, down, up, index, 0.5, want_saved=True)
    dx, dweight, _, ddown, dup = ops.adapter_dense_backward(dy, x, w, None, down, up, index, 0.5, saved=saved, want_dweight=True)
    xd, wd, dd, ud, dyd = (t.double() for t in (x, w, down, up, dy))
    want = {"y": xd @ wd.t(), "dx": dyd @ wd, "ddown": torch.zeros_like(dd), "dup": torch.zeros_like(ud), "dweight": dyd.flatten(0, 1).t() @ xd.flatten(0, 1)}
    for a in range(4):
        r = (index == a).nonzero().view(-1)
        t, dt = 0.5 * xd[r] @ dd[a].t(), 0.5 * dyd[r] @ ud[a]
        want["y"][r] += t @ ud[a].t()
        want["dx"][r] += dt @ dd[a]
        want["ddown"][a] = dt.flatten(0, 1).t() @ xd[r].flatten(0, 1)
        want["dup"][a] = dyd[r].flatten(0, 1).t() @ t.flatten(0, 1)
    for name, got in {"y": y, "dx": dx, "ddown": ddown, "dup": dup, "dweight": dweight}.items():
        assert torch.equal(torch.isfinite(got), torch.isfinite(want[name])), name
        assert torch.isfinite(got).any() and (name == "dweight" or not torch.isfinite(got).all()), name
