"""Rules of the trainable layers' sources, and refusals that need no GPU."""

import re
from pathlib import Path

import pytest
import torch

from bionemo_inference_runtime_b200 import _lib, ops
from bionemo_inference_runtime_b200.csrc import build

CSRC = Path(build.__file__).resolve().parent


def test_matmul_kernel_lets_the_next_kernel_start_behind_its_allocation():
    """The rule of the other tensor-memory kernels, for the one that is a template in a header."""
    text = (CSRC / "matmul.cuh").read_text()
    assert text.count("tmem_alloc(") == 1 and text.count("tmem_alloc_pair(") == 2 and text.count("pdl_trigger()") == 1
    assert re.search(r"tmem_alloc_pair\(.*\);\s*else tmem_alloc\(.*\);\s*if \(.*\) pdl_wait\(\);\s*pdl_trigger\(\);", text)


def test_narrow_kernel_lets_the_next_kernel_start_behind_its_allocation():
    text = (CSRC / "narrow.cuh").read_text()
    assert text.count("tmem_alloc(") == 1 and text.count("pdl_trigger()") == 1
    assert re.search(r"tmem_alloc\(.*\);\s*pdl_trigger\(\);", text)


@pytest.mark.parametrize("header", ["matmul.cuh", "narrow.cuh"])
def test_every_wait_is_bounded(header):
    text = re.sub(r"//[^\n]*", "", (CSRC / header).read_text())
    assert "bar.sync" not in text and "try_wait" not in text and not re.search(r"while\s*\(", text)


def test_entry_points_refuse_before_any_cuda_call():
    with pytest.raises(ValueError, match="NULL"):
        _lib.call("b200ta_layer_norm", None, 8, None, None, 0, None, 8, None, 0, 4, 8, 1e-5, None)
    with pytest.raises(ValueError, match="dtype"):
        _lib.call("b200ta_dense", None, 8, None, 8, None, None, 0, None, 8, None, 0, _lib.DTYPE_F32, 0, 0, 4, 8, 8, None)
    with pytest.raises(ValueError, match="activation"):
        _lib.call("b200ta_dense", None, 8, None, 8, None, None, 0, None, 8, None, 0, 0, 99, 0, 4, 8, 8, None)
    with pytest.raises(ValueError, match="NULL"):
        _lib.call("b200ta_dense_backward", None, 8, None, 8, None, 8, None, None, 0, None, 8, None, None, None, 0, 0, 0, 0, 4, 8, 8, None)
    with pytest.raises(ValueError, match="copies"):
        _lib.call("b200ta_copy_rows", None, 0, None)


def test_host_tensors_and_unknown_activations_are_refused():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.dense(x, w), lambda: ops.gated_dense(x, w), lambda: ops.layer_norm(x),
                 lambda: ops.dense_backward(x, x, w), lambda: ops.gated_dense_backward(x, x, w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="activation"):
        ops.dense(x, w, activation="swish")


def test_activation_codes_are_those_of_the_header():
    text = (CSRC.parent.parent / "include" / "b200ta.h").read_text()
    codes = {k.lower(): int(v) for k, v in re.findall(r"#define B200TA_ACT_(\w+) (\d+)", text)}
    assert codes == ops.ACTIVATIONS
