"""Dropout and adapters without a GPU: sources' rules, refusals before any CUDA call, and the division that finds a row's entry."""

import re
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import bionemo_inference_runtime_b200 as b200
from bionemo_inference_runtime_b200 import _lib, ops
from bionemo_inference_runtime_b200.csrc import build

CSRC = Path(build.__file__).resolve().parent


def test_every_wait_is_bounded():
    for name in ("adapters.cu", "adapters.cuh", "dropout.cu"):
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        assert "bar.sync" not in text and "try_wait" not in text and not re.search(r"while\s*\((?!lanes|\(uint64_t)", text), name


def test_entry_points_refuse_before_any_cuda_call():
    with pytest.raises(ValueError, match="NULL"):
        _lib.call("b200ta_dropout", None, None, None, 0, 1, 1, 8, 100, 1, 0, None, None)
    with pytest.raises(ValueError, match="dtype"):
        _lib.call("b200ta_dropout", 16, None, 16, 7, 1, 1, 8, 100, 1, 0, None, None)
    with pytest.raises(ValueError, match="dropped"):
        _lib.call("b200ta_dropout", 16, None, 16, 0, 1, 1, 8, 65537, 1, 0, None, None)
    with pytest.raises(ValueError, match="sizes"):
        _lib.call("b200ta_dropout", 16, None, 16, 0, 1, 0, 8, 100, 1, 0, None, None)
    with pytest.raises(ValueError, match="multiple"):
        _lib.call("b200ta_dropout", 17, None, 16, 0, 1, 1, 8, 100, 1, 0, None, None)
    with pytest.raises(ValueError, match="NULL"):
        _lib.call("b200ta_adapter_dense", 16, 8, 16, 8, None, None, 0, 16, 8, None, 0, None, None, 0, 0, 0, 4, 8, 8, None)
    with pytest.raises(ValueError, match="activation"):
        _lib.call("b200ta_adapter_dense_backward", 16, 8, 16, 8, 16, 8, None, None, 0, None, None, None, 8, None, None, None, None, None, 0, 0, 99, 0,
                  4, 8, 8, None)


def test_host_tensors_and_bad_probabilities_are_refused():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    down, up = torch.zeros(1, 2, 8, dtype=torch.bfloat16), torch.zeros(1, 6, 2, dtype=torch.bfloat16)
    for call in (lambda: ops.dropout(x, 0.5, 1), lambda: ops.dropout_backward(x, 0.5, 1), lambda: ops.adapter_dense(x, w, None, down, up),
                 lambda: ops.adapter_gated_dense(x, w, None, down, up)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            ops.dropout(x, p, 1)
    with pytest.raises(ValueError, match="axis"):
        ops.dropout(x, 0.5, 1, shared=2)
    with pytest.raises(ValueError, match="activation"):
        ops.adapter_dense(x, w, None, down, up, activation="swish")
    with pytest.raises(ValueError, match="dropout"):
        b200.TrainableTransition(8, 16, dropout=1.5, device="cpu")
    for rank in (-1, 257):
        with pytest.raises(ValueError, match="rank"):
            b200.TrainableTransition(8, 16, adapter_rank=rank, device="cpu")


@pytest.mark.parametrize("function", [b200.adapter_dense, b200.adapter_gated_dense])
def test_derivatives_that_there_are_not_are_refused(function):
    """The gradient of a scale, asked for alone too, and forward-mode derivatives of any argument."""
    x, w, b = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(6)
    down, up, scale = torch.zeros(2, 2, 8), torch.zeros(2, 6, 2), torch.ones(2)
    index = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="scale"):
        function(x, w, b, down, up, index, scale.requires_grad_(True))
    scale.requires_grad_(False)
    with forward_ad.dual_level():
        for k in (0, 1, 2, 3, 4, 6):
            given = [x, w, b, down, up, index, scale]
            given[k] = forward_ad.make_dual(given[k], torch.ones_like(given[k]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                function(*given)
        for k in (0, 1):
            given = [x, x]
            given[k] = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                b200.dropout(given[0], 0.5, 1, residual=given[1])


def test_rows_find_their_entry_by_a_product():
    """n / d = n * ceil(2^(31 + s) / d) >> (31 + s) with 2^s >= d, for n below 2^31: the factor is at most 2^32 - 1 and the quotient exact."""
    divisors = [1, 2, 3, 5, 7, 23, 64, 127, 128, 129, 1000, 36864, 147456, (1 << 30) + 1, (1 << 31) - 1, 1 << 31]
    for d in divisors:
        s = (d - 1).bit_length()
        factor = -(-(1 << (31 + s)) // d)
        assert factor < 1 << 32
        top = (1 << 31) - 1
        near = {k * d + e for k in (0, 1, 2, top // d // 2, top // d - 1, top // d) for e in (-1, 0, 1)} | {top - 1, top}
        for n in (n for n in near if 0 <= n <= top):
            assert n * factor >> (31 + s) == n // d
    assert "((uint64_t(1) << (31 + s)) + d - 1) / d" in (CSRC / "adapters.cuh").read_text()


def test_state_of_an_adapted_transition_merges_into_a_plain_one():
    torch.manual_seed(0)
    layer = b200.TrainableTransition(16, 24, adapter_rank=4, adapters=2, adapter_scale=0.5, device="cpu")
    assert {k for k, p in layer.named_parameters() if p.requires_grad} == {
        f"{n}_adapters.{m}" for n in ("fused_fc2_fc1", "fc3") for m in ("down", "up")}
    plain = b200.TrainableTransition(16, 24, device="cpu")
    assert layer.merged_state_dict(0).keys() == plain.state_dict().keys()
    assert torch.equal(layer.merged_state_dict(1)["fc3.weight"], layer.fc3.weight)  # an adapter begins as nothing
    with torch.no_grad():
        layer.fc3_adapters.up.normal_()
    merged = layer.merged_state_dict(1)["fc3.weight"]
    want = layer.fc3.weight.double() + 0.5 * layer.fc3_adapters.up[1].double() @ layer.fc3_adapters.down[1].double()
    assert torch.equal(merged, want.to(torch.bfloat16))
    assert torch.equal(plain.merged_state_dict()["fc3.weight"], plain.fc3.weight)
    for none in (-1, 2):  # (-1 stands for no adapter elsewhere)
        with pytest.raises(ValueError, match="adapter"):
            layer.merged_state_dict(none)
