"""Infinities in rows and in their gradients: what the formula makes of them, whatever kernels run."""

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
