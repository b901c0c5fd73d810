"""A transition with adapters and dropout, as it is trained and served, and the example that does so."""

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


def randn(*shape, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).bfloat16()


def adapted(dim, hidden, adapters, **more):
    torch.manual_seed(1)
    layer = b200.TrainableTransition(dim, hidden, device=DEV, adapter_rank=12, adapters=adapters, adapter_scale=1.5, **more)
    with torch.no_grad():
        layer.norm.weight.normal_(1, 0.2), layer.norm.bias.normal_(0, 0.2)
        for a in (layer.fused_fc2_fc1_adapters, layer.fc3_adapters):
            a.up.normal_(0, 0.1)
    return layer


def reference(layer, x, index, mask, keep, residual):
    """In 64 bits from the layer's own parameters, request by request, for automatic differentiation."""
    p = {k: v.detach().double().requires_grad_(True) for k, v in layer.named_parameters()}
    xd = x.detach().double().requires_grad_(True)

    def dense(t, name):
        out = []
        for one, g in zip(t, index.tolist(), strict=True):
            z = F.linear(one, p[f"{name}.weight"])
            if 0 <= g < layer.fc3_adapters.down.shape[0]:
                z = z + layer.adapter_scale * F.linear(F.linear(one, p[f"{name}_adapters.down"][g]), p[f"{name}_adapters.up"][g])
            out.append(z)
        return torch.stack(out)

    n = F.layer_norm(xd, (layer.dim,), p["norm.weight"], p["norm.bias"], layer.norm.eps)
    value, gate = dense(n, "fused_fc2_fc1").chunk(2, -1)
    y = dense(value * F.silu(gate), "fc3")
    y = y if mask is None else y * mask.double().unsqueeze(-1)
    y = y if keep is None else y * keep
    return (xd + y if residual else y), xd, p


@pytest.mark.parametrize("dim,hidden,shape", [(128, 512, (4, 24, 24)), (384, 1536, (5, 50)), (72, 100, (6, 7)), (128, 512, (3, 100, 100))])
@pytest.mark.parametrize("masked,residual,drops", [(False, True, True), (True, True, True), (True, False, False), (False, True, False)])
@pytest.mark.parametrize("whole", [False, True])
def test_adapted_transition(dim, hidden, shape, masked, residual, drops, whole):
    """Against the formula in 64 bits, relative to the size of each result: at most ten roundings to bf16 lie between the kernels on the
    way to a gradient (2^-9 each in the root mean square)."""
    layer = adapted(dim, hidden, 3, dropout=0.25 if drops else 0.0, dropout_shared=1)
    if whole:
        layer.requires_grad_(True)
    index = torch.tensor([2, -1, 0, 1, 2, 0][:shape[0]], device=DEV)
    x = randn(*shape, dim, seed=2).requires_grad_(True)
    mask = None if not masked else (torch.rand(*shape, device=DEV) > 0.3).to(torch.bfloat16)
    dy = randn(*shape, dim, seed=3, std=0.1)
    y = layer(x, mask, residual=residual, index=index, seed=77, sequence=3)
    keep = None
    if drops:
        keep = ops.dropout(torch.ones_like(x, dtype=torch.float32), 0.25, 77, 3, shared=1).double()
    want, xd, p = reference(layer, x, index, mask, keep, residual)
    y.backward(dy)
    want.backward(dy.double())
    pairs = {"y": (y, want), "x": (x.grad, xd.grad), **{k: (v.grad, p[k].grad) for k, v in layer.named_parameters() if v.requires_grad}}
    for name, (a, b) in pairs.items():
        assert a.shape == b.shape and ((a.double() - b).norm() / b.norm()).item() < 10 * 2 ** -9, name
    assert whole or all(v.grad is None for k, v in layer.named_parameters() if "_adapters." not in k)


def test_evaluation_drops_nothing_and_seeds_are_drawn():
    layer = adapted(64, 96, 2, dropout=0.5)
    x, index = randn(4, 9, 64, seed=1), torch.tensor([0, 1, -1, 0], device=DEV)
    with torch.no_grad():
        torch.manual_seed(5)
        first, second = layer(x, residual=True, index=index), layer(x, residual=True, index=index)
        assert not torch.equal(first, second)
        torch.manual_seed(5)
        assert torch.equal(first, layer(x, residual=True, index=index))
        assert torch.equal(layer(x, index=index, seed=9), layer(x, index=index, seed=9))
        layer.eval()
        assert torch.equal(layer(x, index=index), layer(x, index=index))
        plain = b200.TrainableTransition(64, 96, device=DEV)
        plain.load_state_dict(layer.merged_state_dict(0), strict=True)
        got, want = layer(x, index=index), plain(x)
        # a request alone, and the weights with its adapter added to them: two bf16 paths
        assert torch.equal(layer(x[:1], index=index[:1]).float().round(decimals=1), got[:1].float().round(decimals=1)) or \
            (layer(x[:1], index=index[:1]) - got[:1]).abs().max() < 2 ** -5
        assert ((got[0] - want[0]).double().norm() / want[0].double().norm()).item() < 10 * 2 ** -9
    with pytest.raises(ValueError, match="adapter"):
        plain(x, index=index)


def test_captured_training_step():
    """Forward and backward captured into a graph (while no eager graph of the same parameters lives: PyTorch's nodes that accumulate
    their gradients would stay on another stream)."""
    layer = adapted(64, 96, 2, dropout=0.2)
    x, dy = randn(4, 50, 64, seed=1), randn(4, 50, 64, seed=2, std=0.1)
    index, seed = torch.tensor([0, 1, -1, 1], device=DEV), torch.tensor([3], device=DEV)
    trained = [p for p in layer.parameters() if p.requires_grad]

    def step():
        y = layer(x, residual=True, index=index, seed=seed)
        return [y.detach(), *torch.autograd.grad(y, trained, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(3):
        seed.fill_(n)
        index.copy_(torch.tensor([n % 2, 1, 0, -1], device=DEV))
        want = step()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want, strict=True))


def test_a_backward_pass_is_not_captured_beside_an_eager_graph_of_its_leaves():
    """Their gradients' nodes lie on the default stream while that graph lives; without it, or with one of another stream, capture works."""
    x, w, dy = randn(32, 64, seed=1), randn(48, 64, seed=2), randn(32, 48, seed=3)
    down, up = (t.requires_grad_(True) for t in (randn(1, 8, 64, seed=4), randn(1, 48, 8, seed=5)))
    want = torch.autograd.grad(b200.adapter_dense(x, w, None, down, up), (down, up), dy)

    def captured():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(b200.adapter_dense(x, w, None, down, up), (down, up), dy)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))

    alive = b200.adapter_dense(x, w, None, down, up)
    with pytest.raises(RuntimeError, match="eager graph"):
        captured()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, (down, up), dy), want, strict=True))
    del alive
    captured()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        alive = b200.adapter_dense(x, w, None, down, up)
    side.synchronize()
    captured()
    del alive


def test_a_captured_step_needs_a_seed():
    layer, x = adapted(64, 96, 2, dropout=0.2), randn(4, 50, 64, seed=1)
    index = torch.tensor([0, 1, -1, 1], device=DEV)
    with torch.no_grad():
        layer(x, index=index)
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()), pytest.raises(ValueError, match="seed"):
            layer(x, index=index)
        layer.eval()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x, index=index)
        graph.replay()
        assert torch.equal(y, layer(x, index=index))


def test_example():
    path = Path(__file__).resolve().parent.parent / "examples" / "finetune_adapters.py"
    spec = importlib.util.spec_from_file_location("finetune_adapters", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, student, apart = example.finetune(tokens=16, steps=3)
    assert len(losses) == 3 and all(loss == loss for loss in losses)
    for name, p in student.named_parameters():
        assert (p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any()) if "_adapters." in name else p.grad is None, name
    assert max(apart) < 0.1  # two bf16 paths of values up to 4
