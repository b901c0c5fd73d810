"""The differentiable functions, the trainable transition and the example that serves what it trained."""

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import bionemo_inference_runtime_b200 as b200
from bionemo_inference_runtime_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    _lib.reset_device_status()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def leaf(*shape, seed, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype).requires_grad_(True)


def test_functions_give_the_gradients_of_the_operators():
    x, w, b, wn, bn = leaf(5, 30, 48, seed=1), leaf(80, 48, seed=2, std=0.15), leaf(80, seed=3), leaf(48, seed=4), leaf(48, seed=5)
    res, dy = leaf(5, 30, 80, seed=6), leaf(5, 30, 80, seed=7).detach()
    y = b200.dense(x, w, b, activation="gelu", residual=res)
    assert torch.equal(y, ops.dense(x, w, b, activation="gelu", residual=res))
    got = torch.autograd.grad(y, (x, w, b, res), dy)
    want = ops.dense_backward(dy, x, w, b, activation="gelu")
    assert all(torch.equal(a, c) for a, c in zip(got, (*want, dy), strict=True))

    dh = dy[..., :40].contiguous()
    y = b200.gated_dense(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dh)
    assert torch.equal(y, ops.gated_dense(x, w, b))
    assert all(torch.equal(a, c) for a, c in zip(got, ops.gated_dense_backward(dh, x, w, b), strict=True))

    dn = dy[..., :48].contiguous()
    y = b200.layer_norm(x, wn, bn, 1e-5)
    got = torch.autograd.grad(y, (x, wn, bn), dn)
    _, stats = ops.layer_norm(x, wn, bn, 1e-5, want_stats=True)
    assert all(torch.equal(a, c) for a, c in zip(got, ops.layer_norm_backward(dn, x, stats, wn), strict=True))


def test_only_inputs_that_need_gradients_get_them():
    x, w, b = leaf(40, 32, seed=1), leaf(64, 32, seed=2), leaf(64, seed=3)
    b200.dense(x.detach(), w, b).sum().backward()
    assert x.grad is None and w.grad is not None and b.grad is not None
    b200.gated_dense(x, w.detach(), b.detach()).sum().backward()  # (the gradient of a sum is broadcast)
    assert x.grad is not None
    with torch.no_grad():
        assert not b200.dense(x, w, b).requires_grad
    res = leaf(40, 64, seed=4)
    b200.dense(x.detach(), w.detach(), None, residual=res).sum().backward()
    assert torch.equal(res.grad, torch.ones_like(res))
    with pytest.raises(RuntimeError):  # first order only
        g = torch.autograd.grad(b200.dense(x, w, b).sum(), x, create_graph=True)[0]
        torch.autograd.grad(g.sum(), x)


def reference(layer, x, mask, residual):
    """The transition in 64 bits from the layer's own parameters, for automatic differentiation."""
    p = {k: v.detach().double().requires_grad_(True) for k, v in layer.named_parameters()}
    xd = x.detach().double().requires_grad_(True)
    n = F.layer_norm(xd, (layer.dim,), p["norm.weight"], p["norm.bias"], layer.norm.eps)
    value, gate = F.linear(n, p["fused_fc2_fc1.weight"]).chunk(2, -1)
    y = F.linear(value * F.silu(gate), p["fc3.weight"])
    y = y if mask is None else y * mask.double().unsqueeze(-1)
    return (xd + y if residual else y), xd, p


@pytest.mark.parametrize("dim,hidden,shape", [(128, 512, (1, 24, 24)), (384, 1536, (2, 50)), (72, 100, (3, 7)), (128, 512, (200, 200))])
@pytest.mark.parametrize("masked,residual", [(False, True), (True, True), (True, False)])
def test_trainable_transition(dim, hidden, shape, masked, residual):
    """Against the formula in 64 bits, relative to the size of each result: the roundings to bf16 between the kernels (2^-9
    each: normalised rows, hidden values, their two gradients, gradient of the normalised rows) add up to less than 8 x 2^-9
    in the root mean square."""
    torch.manual_seed(1)
    layer = b200.TrainableTransition(dim, hidden, device=DEV)
    with torch.no_grad():
        layer.norm.weight.normal_(1, 0.2), layer.norm.bias.normal_(0, 0.2)
    x = leaf(*shape, dim, seed=2)
    mask = None if not masked else (torch.rand(*shape, device=DEV) > 0.3).to(torch.bfloat16)
    dy = leaf(*shape, dim, seed=3, std=0.1).detach()
    y = layer(x, mask, residual=residual)
    want, xd, p = reference(layer, x, mask, residual)
    y.backward(dy)
    want.backward(dy.double())
    pairs = {"y": (y, want), "x": (x.grad, xd.grad), **{k: (v.grad, p[k].grad) for k, v in layer.named_parameters()}}
    for name, (a, b) in pairs.items():
        assert a.shape == b.shape and ((a.double() - b).norm() / b.norm()).item() < 8 * 2 ** -9, name


def test_trained_weights_serve():
    path = Path(__file__).resolve().parent.parent / "examples" / "finetune_transition.py"
    spec = importlib.util.spec_from_file_location("finetune_transition", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, apart = example.finetune(tokens=24, steps=40)
    assert losses[-1] < 0.5 * losses[0]
    assert apart < 0.1  # two bf16 paths of values up to 4


def test_refusals():
    with pytest.raises(ValueError):
        b200.TrainableTransition(16, 32, dtype=torch.float32)
    with pytest.raises(ValueError):
        b200.TrainableTransition(16, 32, out_dim=24)(leaf(4, 16, seed=1), residual=True)
    with pytest.raises(ValueError):
        b200.TrainableTransition(16, 32)(leaf(4, 24, seed=1))
