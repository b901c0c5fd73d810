"""Backward passes captured into a graph beside an eager graph whose gradients are accumulated on the default stream."""

import pytest
import torch

import bionemo_inference_runtime_b200 as b200

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).bfloat16()


def captured(step):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
def test_only_gradients_that_are_asked_for_count(gated):
    """A captured backward pass that has nothing to add to the eager graph's leaves is captured, and right."""
    function = b200.adapter_gated_dense if gated else b200.adapter_dense
    w, dy = randn(96 if gated else 48, 64, seed=2), randn(32, 48, seed=3)
    down, up = (t.requires_grad_(True) for t in (randn(1, 8, 64, seed=4), randn(1, w.shape[0], 8, seed=5)))
    given = randn(32, 64, seed=1)
    x = given.clone().requires_grad_(True)
    want = torch.autograd.grad(function(x, w, None, down, up), x, dy)[0]
    del x
    alive = function(given, w, None, down, up)  # holds the nodes of down and up
    x = given.clone().requires_grad_(True)
    assert torch.equal(captured(lambda: torch.autograd.grad(function(x, w, None, down, up), x, dy)[0]), want)
    assert alive.requires_grad


def functions():
    """Every differentiable function of its tensors, and those tensors."""
    x, w, gates, bias, n = randn(32, 64, seed=1), randn(48, 64, seed=2), randn(96, 64, seed=3), randn(48, seed=4), randn(64, seed=5)
    down, up, up2, r = randn(1, 8, 64, seed=6), randn(1, 48, 8, seed=7), randn(1, 96, 8, seed=8), randn(32, 48, seed=9)
    return {
        "layer_norm": (lambda x, n, b: b200.layer_norm(x, n, b), (x, n, n.flip(0))),
        "dense": (lambda x, w, b, r: b200.dense(x, w, b, activation="silu", residual=r), (x, w, bias, r)),
        "gated_dense": (lambda x, w, b: b200.gated_dense(x, w, b), (x, gates, bias.repeat(2))),
        "adapter_dense": (lambda x, w, b, d, u, r: b200.adapter_dense(x, w, b, d, u, residual=r), (x, w, bias, down, up, r)),
        "adapter_gated_dense": (lambda x, w, b, d, u: b200.adapter_gated_dense(x, w, b, d, u), (x, gates, bias.repeat(2), down, up2)),
        "dropout": (lambda x, r: b200.dropout(x, 0.3, 5, residual=r), (r, r.flip(0))),
    }


@pytest.mark.parametrize("name", ["layer_norm", "dense", "gated_dense", "adapter_dense", "adapter_gated_dense", "dropout"])
def test_each_leaf_is_refused_by_name_and_captured_without_the_eager_graph(name):
    function, given = functions()[name]
    dy = randn(*function(*given).shape, seed=20)
    for i in range(len(given)):  # one argument is a leaf at a time
        leaf = given[i].clone().requires_grad_(True)
        args = [leaf if j == i else t for j, t in enumerate(given)]
        step = lambda: torch.autograd.grad(function(*args), leaf, dy)[0]  # noqa: B023, E731
        want = step()
        alive = function(*args)
        for refused in (step, lambda: function(*args).backward(dy)):  # noqa: B023
            with pytest.raises(RuntimeError, match="eager graph"):
                captured(refused)
        assert torch.equal(torch.autograd.grad(alive, leaf, dy)[0], want)
        del alive
        assert torch.equal(captured(step), want), i
