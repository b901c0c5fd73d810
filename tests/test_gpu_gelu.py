"""gelu by itself: products with a single term are exact, so what is off is the activation's, or the result's rounding."""

import pytest
import torch

from bionemo_inference_runtime_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def formula(z):
    """gelu(z) and its slope, by erfc, which does not cancel below zero; p(-|z|) and z times the density."""
    tail = 0.5 * torch.erfc(z.abs() * 0.5 ** 0.5)
    p = torch.where(z < 0, tail, 1 - tail)
    peak = z * torch.exp(-0.5 * z * z) * (0.5 / torch.pi) ** 0.5
    return z * p, p + peak, tail, peak


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_gelu_alone(rows, dtype):
    """The approximation of p is within 7.5e-8; the products and sums behind it are ten or so, of values with p(-|z|) as a factor
    (2^-19 of it) and one with 1 (2^-24).  The result is rounded once, its gradient before the activation once and its sum again."""
    z = torch.linspace(-8, 8, 4001, device=DEV).to(dtype)
    x, w = torch.zeros(rows, 8, device=DEV, dtype=dtype), torch.zeros(z.numel(), 8, device=DEV, dtype=dtype)
    x[:, 3], w[:, 3] = 1, z
    value, slope, tail, peak = formula(z.double())
    p_bound = 0.75e-7 + 2.0 ** -19 * tail + 2.0 ** -24
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    y = ops.dense(x, w, activation="gelu").double()
    assert ((y - value).abs() <= 1.01 * half * value.abs() + z.double().abs() * p_bound + tiny).all()
    dy = torch.zeros(rows, z.numel(), device=DEV, dtype=dtype)
    dy[-1] = 1
    db = ops.dense_backward(dy, x, w, activation="gelu", want_dx=False, want_dweight=False, want_dbias=True)[2].double()
    assert ((db - slope).abs() <= 2.02 * half * slope.abs() + p_bound + 2.0 ** -19 * peak.abs() + 2 * tiny).all()
