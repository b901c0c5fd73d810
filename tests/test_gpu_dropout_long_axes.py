"""Dropout beside shared axes so long that a thread takes their entries in several rounds.

An entry of the shared axis has the draw of a tensor that consists of it alone, which the small tests compare with the generator's
definition: the results are equal bit by bit."""

import pytest
import torch

from bionemo_inference_runtime_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (outer, axis, inner): whole vectors, odd rows of several windows and of a part of one, and the elements one by one
SHAPES = [(1, 512, 65536), (3, 700, 16384), (60, 100, 5001), (400, 1000, 41), (64, 512, 2049), (3000, 513, 1), (900, 300, 7)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_each_entry_has_the_draw_of_the_axis(shape, dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    x, r = (torch.randn(*shape, generator=g, device=DEV, dtype=dtype) for _ in range(2))
    keep = ops.dropout(torch.ones(shape[0], 1, shape[2], device=DEV), 0.3, 5, 9) != 0
    for residual in (None, r):
        y = ops.dropout(x, 0.3, 5, 9, residual=residual, shared=1)
        base = torch.zeros_like(x) if residual is None else residual
        assert torch.equal(torch.where(keep, base, y), base)
        for a in {0, 1, 3, 4, 7, shape[1] // 2, shape[1] - 2, shape[1] - 1}:
            one = ops.dropout(x[:, a].contiguous(), 0.3, 5, 9, residual=None if residual is None else r[:, a].contiguous())
            assert torch.equal(y[:, a], one)
        # all entries at once: x / (1 - p) in 64 bits, with the two roundings of 32 bits and the last one
        term = x.double() * keep / (1 - round(0.3 * 65536) / 65536)
        want = term + base.double()
        bound = 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -22 * (term.abs() + base.double().abs()) + torch.finfo(dtype).smallest_normal
        assert ((y.double() - want).abs() <= bound).all()
