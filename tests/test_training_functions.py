"""What the differentiable functions ask for and refuse, on the CPU with plain stand-ins for the kernels."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import bionemo_inference_runtime_b200 as b200
from bionemo_inference_runtime_b200.layers import training


@pytest.fixture
def kernels(monkeypatch):
    """Plain forward passes in the operators' places; returns the calls' keyword arguments."""
    calls = []

    def dense(x, weight, bias=None, *, activation="none", residual=None, want_saved=False):
        calls.append({"want_saved": want_saved})
        y = x @ weight.t() if bias is None else x @ weight.t() + bias
        y = y if residual is None else y + residual
        return (y, None) if want_saved else y

    def gated_dense(x, weight, bias=None, *, activation="silu", want_saved=False):
        calls.append({"want_saved": want_saved})
        value, gate = (x @ weight.t()).chunk(2, -1)
        return (value * gate, None) if want_saved else value * gate

    def layer_norm(x, weight=None, bias=None, eps=1e-5, *, want_stats=False):
        calls.append({"want_stats": want_stats})
        return (x, x.new_zeros(x.shape[0], 2)) if want_stats else x

    for f in (dense, gated_dense, layer_norm):
        monkeypatch.setattr(training.ops, f.__name__, f)
    return calls


FUNCTIONS = {
    "dense": lambda x, w, b, r: b200.dense(x, w, b, residual=r),
    "gated_dense": lambda x, w, b, r: b200.gated_dense(x, w, b),
    "layer_norm": lambda x, w, b, r: b200.layer_norm(x, w[0], b[:4]),
}


@pytest.mark.parametrize("name", list(FUNCTIONS))
def test_forward_mode_is_refused(kernels, name):
    """A result without a tangent would say that it does not depend on its inputs."""
    x, w, b, r = torch.randn(3, 4), torch.randn(6, 4), torch.randn(6), torch.randn(3, 6)
    takes = 4 if name == "dense" else 3
    with forward_ad.dual_level():
        assert not FUNCTIONS[name](x, w, b, r).requires_grad  # tensors without a tangent pass
        for k in range(takes):
            given = [x, w, b, r]
            given[k] = forward_ad.make_dual(given[k], torch.ones_like(given[k]))
            for on in (True, False):
                with torch.set_grad_enabled(on), pytest.raises(NotImplementedError, match="forward-mode"):
                    FUNCTIONS[name](*given)
    assert not FUNCTIONS[name](x, w, b, r).requires_grad


def test_nothing_is_kept_for_gradients_that_do_not_need_it(kernels):
    """The gradient of a residual is dy: where only that is wanted, the values before the activation are not kept."""
    x, w, b, r = torch.randn(3, 4), torch.randn(6, 4), torch.randn(6), torch.randn(3, 6)
    y = b200.dense(x, w, b, activation="gelu", residual=r.requires_grad_(True))
    assert kernels.pop() == {"want_saved": False} and y.requires_grad
    y.sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))
    for needs in (x, w, b):
        needs.requires_grad_(True)
        b200.dense(x, w, b, activation="gelu", residual=r)
        assert kernels.pop() == {"want_saved": True}
        needs.requires_grad_(False)
