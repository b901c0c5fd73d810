"""Dropout against its definition: Philox in Python integers, sums in 64 bits.

Tolerances: the factor 65536 / (65536 - d) and the fused product and sum are off by two roundings of 32 bits (2^-24 each of their terms),
the result by one rounding to its type; what is dropped is the residual, bit by bit.
"""

import math

import pytest
import torch

import bionemo_inference_runtime_b200 as b200
from bionemo_inference_runtime_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
M32 = (1 << 32) - 1


def philox(block: int, sequence: int, seed: int) -> list[int]:
    c = [block & M32, block >> 32, sequence & M32, sequence >> 32]
    k = [seed & M32, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & M32, (a >> 32) ^ c[3] ^ k[1], a & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def test_philox_is_the_published_generator():
    """The known answers of the generator's authors for counters and keys of zeros, of ones, and of digits of pi."""
    assert philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert philox(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox(0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def keep_of(shape, p, seed, sequence, shared):
    """The elements that stay, as [outer, 1 or axis, inner] of booleans broadcast to the shape."""
    drawn = [1 if d == shared else n for d, n in enumerate(shape)]
    dropped, kept = round(p * 65536), []
    for block in range((math.prod(drawn) + 7) // 8):
        for word in philox(block, sequence, seed):
            kept += [(word & 0xFFFF) >= dropped, (word >> 16) >= dropped]
    return torch.tensor(kept[:math.prod(drawn)], device=DEV).view(drawn).expand(shape), dropped


def check(x, p, seed, sequence=0, residual=None, shared=None, out=None):
    axis = None if shared is None else shared % x.dim()
    keep, dropped = keep_of(tuple(x.shape), p, seed % (1 << 64), sequence, axis)
    got = ops.dropout(x, p, seed, sequence, residual=residual, shared=shared, out=out)
    base = torch.zeros_like(x) if residual is None else residual
    assert torch.equal(got[~keep], base[~keep])
    if keep.any():
        term = x[keep].double() / (1 - dropped / 65536)
        want = term + base[keep].double()
        bound = 1.01 * torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0 ** -22 * (term.abs() + base[keep].double().abs()) + torch.finfo(x.dtype).smallest_normal
        assert ((got[keep].double() - want).abs() <= bound).all()
    return got


def randn(*shape, seed, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


# around whole vectors, a thread's eight elements and the windows of 2040 elements that odd rows are taken in
SHAPES = [(1,), (7,), (8,), (9, 1), (5, 3), (3, 16), (2, 3, 17), (2, 7, 8), (3, 5, 100), (2, 9, 127), (2, 3, 2039), (1, 5, 2041), (2, 3, 4099),
          (60, 2, 24), (4, 1, 31)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_dropout(shape, dtype):
    x, residual = randn(*shape, seed=1, dtype=dtype), randn(*shape, seed=2, dtype=dtype)
    for i, shared in enumerate([None, *range(len(shape))]):
        check(x, 0.3, 1234567890123 + i, 5 + i, shared=shared)
        check(x, 0.61, -7, (1 << 40) + 3, residual=residual, shared=shared)


@pytest.mark.parametrize("p", [0.0, 1.0, 2.0 ** -17, 0.5, 65535.4 / 65536])
@pytest.mark.parametrize("shape,shared", [((40, 100), None), ((4, 10, 24), 1), ((4, 10, 25), 1)])
def test_probabilities(p, shape, shared):
    x = randn(*shape, seed=1, dtype=torch.float32)
    check(x, p, 99, shared=shared)
    check(x, p, 99, residual=randn(*shape, seed=2, dtype=torch.float32), shared=shared)
    if p == 0:
        assert torch.equal(ops.dropout(x, p, 99, shared=shared), x)


def test_share_of_what_is_dropped():
    """Of n independent draws a share p is dropped, to five standard deviations."""
    n, p = 1 << 24, 0.15
    y = ops.dropout(torch.ones(n, device=DEV), p, 3)
    assert abs((y == 0).double().mean().item() - p) < 5 * math.sqrt(p * (1 - p) / n) + 2.0 ** -17
    other = ops.dropout(torch.ones(n, device=DEV), p, 3, 1)
    both = ((y == 0) & (other == 0)).double().mean().item()  # another sequence is another draw
    assert abs(both - p * p) < 5 * math.sqrt(p * p / n) + 2.0 ** -17


@pytest.mark.parametrize("shared", [None, 0, 1])
def test_dropped_infinities_and_nan_vanish(shared):
    x, residual = randn(6, 8, 40, seed=1), randn(6, 8, 40, seed=2)
    keep, _ = keep_of((6, 8, 40), 0.4, 11, 0, shared)
    bad = torch.where(keep, x, torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=DEV).bfloat16().repeat(480).view(6, 8, 40))
    for r in (None, residual):
        assert torch.equal(ops.dropout(bad, 0.4, 11, residual=r, shared=shared), ops.dropout(x, 0.4, 11, residual=r, shared=shared))


def test_strides_and_places():
    base, wide = randn(6, 5, 3, 160, seed=1), randn(3000, seed=4)
    for x in (base[..., 7:107], base.transpose(0, 2), base[:, 1:4, :, ::2], base[:1].expand(4, 5, 3, 160), base.permute(0, 1, 3, 2)):
        r = randn(*x.shape, seed=2)
        for shared in (None, 1):
            want = ops.dropout(x.contiguous(), 0.3, 5, residual=r, shared=shared)
            assert torch.equal(ops.dropout(x, 0.3, 5, residual=r, shared=shared), want)
    for first in (1, 3, 8):  # addresses off the 16-byte boundaries
        for shape, shared in (((10, 96), None), ((5, 12, 16), 1), ((5, 12, 15), 1)):
            x = wide[first:first + math.prod(shape)].view(shape)
            check(x, 0.3, 5, shared=shared)
            held = torch.full((math.prod(shape) + 16,), 7.0, device=DEV, dtype=torch.bfloat16)
            out = held[first:first + math.prod(shape)].view(shape)
            assert torch.equal(ops.dropout(x, 0.3, 5, shared=shared, out=out), ops.dropout(x.clone(), 0.3, 5, shared=shared))
            assert (held[:first] == 7).all() and (held[first + math.prod(shape):] == 7).all()
    assert ops.dropout(base[:0], 0.3, 5).shape == (0, 5, 3, 160)


def test_out_may_be_what_is_read_itself():
    x, r = randn(30, 50, seed=1), randn(30, 50, seed=2)
    want = ops.dropout(x, 0.3, 5, residual=r)
    for out in (x.clone(), r.clone()):
        a, b = (out, r) if torch.equal(out, x) else (x, out)
        assert ops.dropout(a, 0.3, 5, residual=b, out=out).data_ptr() == out.data_ptr() and torch.equal(out, want)
    held = randn(31, 50, seed=3)
    for call in (lambda: ops.dropout(held[:30], 0.3, 5, out=held[1:]), lambda: ops.dropout(x, 0.3, 5, residual=held[:30], out=held[1:]),
                 lambda: ops.dropout(x, 0.3, 5, out=held[:30].t().contiguous().t()), lambda: ops.dropout(x, 0.3, 5, out=held)):
        with pytest.raises(ValueError, match="out"):
            call()


def test_refusals():
    x = randn(4, 8, seed=1)
    for call, word in ((lambda: ops.dropout(x, 0.5, 1, residual=x[:2]), "residual"), (lambda: ops.dropout(x, 0.5, 1, residual=x.float()), "residual"),
                       (lambda: ops.dropout(x.int(), 0.5, 1), "x must"), (lambda: ops.dropout(x, 0.5, torch.ones(2, device=DEV, dtype=torch.long)), "seed"),
                       (lambda: ops.dropout(x, 0.5, torch.ones(1, device=DEV)), "seed"), (lambda: ops.dropout(x, 0.5, torch.ones(1).long()), "seed"),
                       (lambda: ops.dropout(x[0, 0], 0.5, 1), "axis")):
        with pytest.raises(ValueError, match=word):
            call()


def test_gradients():
    """The gradient of the function is the function of the gradient; differences in 64 bits are exact, since it is linear."""
    x, r, dy = (randn(7, 12, 40, seed=s, dtype=torch.float32) for s in (1, 2, 3))
    for shared in (None, 0, -2):
        a, b = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
        y = b200.dropout(a, 0.25, 17, 4, residual=b, shared=shared)
        assert torch.equal(y, ops.dropout(x, 0.25, 17, 4, residual=r, shared=shared))
        dx, dr = torch.autograd.grad(y, (a, b), dy)
        assert torch.equal(dx, ops.dropout(dy, 0.25, 17, 4, shared=shared)) and torch.equal(dr, dy)
        step = ops.dropout(x + dy, 0.25, 17, 4, shared=shared).double() - ops.dropout(x, 0.25, 17, 4, shared=shared).double()
        assert ((step - dx.double()).abs() <= 2.0 ** -20 * (x.abs() + dy.abs()).double()).all()
    a = x.clone().requires_grad_(True)
    b200.dropout(a, 0.25, 17).sum().backward()  # (the gradient of a sum is broadcast)
    assert torch.equal(a.grad, ops.dropout(torch.ones_like(x), 0.25, 17))
    with torch.no_grad():
        assert not b200.dropout(a, 0.25, 17).requires_grad
    with pytest.raises(RuntimeError):  # first order only
        g = torch.autograd.grad(b200.dropout(a, 0.25, 17).square().sum(), a, create_graph=True)[0]
        torch.autograd.grad(g.sum(), a)


def test_a_seed_on_the_device_is_read_at_each_replay():
    x, r = randn(50, 64, seed=1), randn(50, 64, seed=2)
    seed, out = torch.tensor([5], device=DEV), torch.empty_like(x)
    assert torch.equal(ops.dropout(x, 0.3, seed, residual=r), ops.dropout(x, 0.3, 5, residual=r))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.dropout(x, 0.3, seed, 9, residual=r, out=out)
        seed += 1
    for n in range(3):
        graph.replay()
        assert torch.equal(out, ops.dropout(x, 0.3, 5 + n, 9, residual=r))
    a = x.clone().requires_grad_(True)
    y = b200.dropout(a, 0.3, seed)
    seed += 100  # the backward pass drops what the forward pass did
    y.backward(r)
    assert torch.equal(a.grad, ops.dropout(r, 0.3, 8))


def test_other_streams():
    x = randn(512, 1024, seed=1)
    want = ops.dropout(x * 2, 0.3, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.dropout(x * 2, 0.3, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
