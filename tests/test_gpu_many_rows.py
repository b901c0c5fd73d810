"""Dense layers of more rows than a grid's second axis has places for blocks of them."""

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


@pytest.mark.parametrize("rows", [65535 * 1024, 65535 * 1024 + 1, 65535 * 1024 + 5000])
def test_bias_gradient_of_many_rows(rows):
    """db alone, of a layer without an activation (which is not cut into chunks): values at both ends and in the middle, whose
    sums are exact."""
    dy = torch.zeros(rows, 8, device=DEV, dtype=torch.bfloat16)
    x, w = torch.zeros(1, 8, device=DEV, dtype=torch.bfloat16).expand(rows, 8), torch.zeros(8, 8, device=DEV, dtype=torch.bfloat16)
    for n, row in enumerate((0, 1, 1023, 1024, rows // 2, 65534 * 1024, 65535 * 1024 - 1, rows - 1)):
        dy[row, n] += 3
        dy[row, 0] += 1
    want = torch.full((8,), 3.0)
    want[0] += 8
    db = ops.dense_backward(dy, x, w, want_dx=False, want_dweight=False, want_dbias=True)[2]
    assert torch.equal(db.float().cpu(), want)
