"""Results written to a tensor of the caller's."""

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


def randn(*shape, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


@pytest.mark.parametrize("rows", [5, 90])
def test_rows_that_lie_on_one_another_are_refused(rows):
    x, w = randn(rows, 48, seed=1), randn(96, 48, seed=2, std=0.1)
    for width, call in ((48, lambda out: ops.layer_norm(x, out=out)), (96, lambda out: ops.dense(x, w, out=out)),
                        (48, lambda out: ops.gated_dense(x, w, out=out))):
        held = torch.zeros(rows * width, device=DEV, dtype=x.dtype)
        for stride in (0, 1, width - 8):
            with pytest.raises(ValueError, match="overlap itself"):
                call(held.as_strided((rows, width), (stride, 1)))
        with pytest.raises(ValueError):
            call(held[:rows].view(rows, 1).expand(rows, width))
        assert not held.any()
        call(held.view(rows, width))
        assert held.any()
