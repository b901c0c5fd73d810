"""Results written to a tensor of the caller's."""

import pytest
import torch

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


@pytest.mark.parametrize("rows", [5, 90])
def test_results_over_what_is_read_are_refused(rows):
    held = randn(rows + 1, 96, seed=1)
    x, square, wide = held[:rows, :48], randn(49, 48, seed=2, std=0.1)[:48], randn(96, 48, seed=3, std=0.1)
    kept = held.clone()
    for name, call in (("x", lambda: ops.dense(x, square, out=x)), ("x", lambda: ops.gated_dense(x, wide, out=x)),
                       ("x", lambda: ops.dense(x, square, out=held[1:, :48])), ("x", lambda: ops.dense(x, square, out=held[:rows, 40:88])),
                       ("x", lambda: ops.layer_norm(x, out=held[1:, :48])), ("x", lambda: ops.layer_norm(x, out=held[:rows, 8:56])),
                       ("residual", lambda: ops.dense(randn(rows, 48, seed=4), square, residual=x, out=held[1:, :48]))):
        with pytest.raises(ValueError, match=f"overlap {name}"):
            call()
        assert torch.equal(held, kept)
    w = randn(48, 48, seed=5, std=0.1)
    with pytest.raises(ValueError, match="overlap weight"):
        ops.dense(w[:5], w, out=w[40:45])
    both = randn(48 + rows * 48, seed=6)
    for call in (lambda out: ops.dense(x, square, both[:48], out=out), lambda out: ops.layer_norm(x, square[0], both[:48], out=out)):
        with pytest.raises(ValueError, match="overlap bias"):
            call(both[24:24 + rows * 48].view(rows, 48))
    with pytest.raises(ValueError, match="overlap weight"):
        ops.layer_norm(x, both[:48], out=both[24:24 + rows * 48].view(rows, 48))


@pytest.mark.parametrize("rows,width", [(5, 48), (90, 48), (90, 51), (700, 4100)])
def test_results_beside_what_is_read_and_in_its_place(rows, width):
    """Columns beside those that are read, the very rows that a layer norm or a residual reads, and rows that are copied first."""
    w, norm = randn(width, width, seed=2, std=width ** -0.5), randn(width, seed=3)
    held = randn(rows, 2 * width, seed=1)
    copy, room = held.clone(), torch.empty_like(held)  # laid out alike: a layer norm's sums go by the boundaries of its rows
    x, beside, kept = held[:, :width], held[:, width:], copy[:, :width]
    want = ops.dense(kept, w, activation="silu", out=room[:, width:])
    ops.dense(x, w, activation="silu", out=beside)
    assert torch.equal(beside, want) and torch.equal(x, kept)
    want = ops.layer_norm(kept, norm, out=room[:, width:])
    ops.layer_norm(x, norm, out=beside)
    assert torch.equal(beside, want) and torch.equal(x, kept)
    want = ops.layer_norm(kept, norm, norm, out=room[:, :width])
    ops.layer_norm(x, norm, norm, out=x)
    assert torch.equal(x, want)
    other = randn(rows, width, seed=4)
    want = ops.dense(other, w, residual=x)
    ops.dense(other, w, residual=x, out=x)
    assert torch.equal(x, want)
    swapped = randn(width, rows, seed=5).t()
    want = ops.dense(swapped, w)
    out = torch.as_strided(swapped, (rows, width), (width, 1))  # the memory of x, which is copied first since its columns lie apart
    ops.dense(swapped, w, out=out)
    assert torch.equal(out, want)


def test_a_result_over_what_a_backward_pass_needs_is_noticed():
    """Automatic differentiation goes by a tensor's version: a result that is written to it counts as a change."""
    w, norm = randn(64, 48, seed=2, std=0.1).requires_grad_(True), randn(48, seed=3)
    z, square = randn(90, 48, seed=4), randn(48, 48, seed=5, std=0.1)
    for call in (lambda out: ops.layer_norm(z, norm, out=out), lambda out: ops.dense(z, square, out=out),
                 lambda out: ops.gated_dense(z, torch.cat([square, square]), out=out)):
        x = randn(90, 48, seed=1)
        loss = b200.dense(x, w, activation="silu").float().sum()
        call(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        x = torch.empty_like(z)
        assert torch.equal(ops.layer_norm(z, norm, out=x), ops.layer_norm(z, norm))
