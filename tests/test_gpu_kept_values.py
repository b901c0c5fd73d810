"""Pre-activations that a dense layer's forward pass keeps for its backward pass, and what the backward pass makes of them."""

import pytest
import torch

from bionemo_inference_runtime_b200 import _lib, ops

from .test_gpu_trainable import half_spacing, layer_formula, layer_inputs, within

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM = 2.0 ** -18  # of the sum of the absolute terms: sums of up to a few thousand terms in 32 bits


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    _lib.reset_device_status()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def randn(*shape, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def padded(n):
    return (n + 7) // 8 * 8


@pytest.mark.parametrize("gated", [False, True], ids=["dense", "gated"])
@pytest.mark.parametrize("rows,K,N,first,pitch", [(4000, 1536, 1283, 0, 1283), (4000, 1536, 1280, 3, 1280), (9000, 1600, 70, 0, 70),
                                                  (2100, 2048, 2047, 5, 2055)])
def test_kept_values_beside_results_that_are_stored_in_place(rows, K, N, first, pitch, gated):
    """Results that a TMA store cannot address (`first` elements off a boundary, rows `pitch` apart) leave row by row, between the
    bulk stores of the kept values: these are the formula's, and the same bits as beside results that TMA takes."""
    columns = 2 * N if gated else N
    x, w, bias = randn(rows, K, seed=1), randn(columns, K, seed=2, std=K ** -0.5), randn(columns, seed=3, std=0.3)
    layer = ops.gated_dense if gated else ops.dense
    aligned = torch.empty(rows, padded(N), device=DEV, dtype=x.dtype)[:, :N]
    y, kept = layer(x, w, bias, activation="gelu", want_saved=True, out=aligned)
    z, size = x.double() @ w.double().t() + bias.double(), x.double().abs() @ w.double().abs().t() + bias.double().abs()
    for part in range(2 if gated else 1):
        got = kept[:, part * padded(N):][:, :N].double()
        at = slice(part * N, (part + 1) * N)
        assert ((got - z[:, at]).abs() <= SUM * size[:, at]).all()
    for _ in range(4):
        held = torch.empty(first + rows * pitch, device=DEV, dtype=x.dtype)
        out = held[first:].as_strided((rows, N), (pitch, 1))
        again, kept_again = layer(x, w, bias, activation="gelu", want_saved=True, out=out)
        assert torch.equal(again, y)
        for part in range(2 if gated else 1):
            at = slice(part * padded(N), part * padded(N) + N)
            assert torch.equal(kept_again[:, at], kept[:, at])


def backward(dy, x, w, bias, saved, activation, gated, want, held):
    """The C entry point on a workspace inside `held`, whose rest is looked at by the caller; returns dx, dW, db and its size."""
    rows, K = x.shape
    N = dy.shape[1]
    outer, code = 2 if gated else 1, ops.ACTIVATIONS[activation]
    need = _lib.load().b200ta_dense_backward_workspace_bytes(code, gated, saved is not None, want[2], rows, K, N)
    assert need <= held.numel()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(outer * N, device=DEV, dtype=x.dtype)
    dx_p, dw_p, db_p = (t.data_ptr() if on else None for t, on in zip((dx, dw, db), want, strict=True))
    _lib.call("b200ta_dense_backward", dy.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, None if bias is None else bias.data_ptr(),
              None if saved is None else saved.data_ptr(), 0 if saved is None else saved.stride(0), dx_p, K, dw_p, db_p, held.data_ptr(), need,
              _lib.DTYPE_BF16, code, gated, rows, K, N, torch.cuda.current_stream().cuda_stream)
    return dx, dw, db, need


@pytest.mark.parametrize("rows,K,N", [(300, 64, 72), (5000, 64, 640), (700, 2048, 2048)])
@pytest.mark.parametrize("want", [(1, 1, 1), (0, 1, 1), (0, 0, 1), (1, 0, 1)])
def test_kept_values_of_a_layer_without_an_activation(rows, K, N, want):
    """Its dz is dy and kept values are not read: with them, on a workspace full of NaN, all gradients are those without."""
    x, w, dy = randn(rows, K, seed=1), randn(N, K, seed=2, std=K ** -0.5), randn(rows, N, seed=3, std=0.1)
    saved = randn(rows, N, seed=4, dtype=torch.float32)
    held = torch.full((1 << 25,), float("nan"), device=DEV).view(torch.uint8)
    with_saved = backward(dy, x, w, None, saved, "none", False, want, held)[:3]
    without = backward(dy, x, w, None, None, "none", False, want, held)[:3]
    for a, b in zip(with_saved, without, strict=True):
        assert torch.equal(a, b)
    db = ops.dense_backward(dy, x, w, saved=saved, want_dx=bool(want[0]), want_dweight=bool(want[1]), want_dbias=True)[2]
    assert torch.equal(db, with_saved[2])


def forward_kept(x, w, bias, activation, gated):
    """The pre-activations by the C entry point, which gives them for any width."""
    rows, K = x.shape
    outer = 2 if gated else 1
    N = w.shape[0] // outer
    y = torch.empty(rows, N, device=DEV, dtype=x.dtype)
    saved = torch.full((rows, outer * padded(N)), float("nan"), device=DEV)
    _lib.call("b200ta_dense", x.data_ptr(), K, w.data_ptr(), K, bias.data_ptr(), None, 0, y.data_ptr(), N, saved.data_ptr(), saved.shape[1],
              _lib.DTYPE_BF16, ops.ACTIVATIONS[activation], gated, rows, K, N, torch.cuda.current_stream().cuda_stream)
    return saved


def check_gradients(got, want, x, w, bias, dy, activation, gated):
    """dx, dW and db (those that were wanted) against the formulas in 64 bits: dz is rounded between the kernels."""
    u, tiny = half_spacing(x.dtype), torch.finfo(x.dtype).smallest_normal
    _, _, dz, sums = layer_formula(x, w, bias, None, activation, gated, dy)
    off = SUM * sums + 1.01 * u * dz.abs() + tiny
    xd, wd = x.double(), w.double()
    for k, (name, exact, bound) in enumerate((("dx", lambda: dz @ wd, lambda: off @ wd.abs() + SUM * (dz.abs() @ wd.abs())),
                                              ("dW", lambda: dz.t() @ xd, lambda: off.t() @ xd.abs() + SUM * (dz.abs().t() @ xd.abs())),
                                              ("db", lambda: dz.sum(0), lambda: off.sum(0) + SUM * dz.abs().sum(0)))):
        if want[k]:
            result = exact()
            within(got[k], result, 1.01 * u * result.abs() + bound() + tiny, name)


CHOICES = [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)]


@pytest.mark.parametrize("rows,K,N,gated", [(1000, 104, 1000, True), (3000, 64, 640, False), (300, 1600, 264, True), (2047, 520, 1288, False)])
def test_the_workspace_of_kept_values_is_enough_for_every_choice_of_gradients(rows, K, N, gated):
    """Kept values give db on the way, a row of sums for each block of rows: nothing lies behind the workspace for any choice."""
    given = layer_inputs(rows, K, N, torch.bfloat16, gated, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    saved = forward_kept(x, w, bias, "gelu", gated)
    held = torch.empty(256 << 20, device=DEV, dtype=torch.uint8)
    for want in CHOICES:
        held.fill_(0xFF)  # (as numbers: NaN)
        *got, need = backward(dy, x, w, bias, saved, "gelu", gated, want, held)
        assert (held[need:] == 0xFF).all(), want
        for t, on in zip(got, want, strict=True):
            assert on or not t.any(), want
        check_gradients(got, want, x, w, bias, dy, "gelu", gated)


@pytest.mark.parametrize("rows,K,N,gated,want", [(250001, 64, 1024, True, (1, 1, 1)), (250001, 64, 1024, True, (0, 0, 1)),
                                                 (300001, 24, 1000, False, (0, 1, 1))])
def test_kept_values_in_chunks(rows, K, N, gated, want):
    """More than half a gigabyte of dz: the backward pass takes the rows in several chunks, the last one a shorter one."""
    given = layer_inputs(rows, K, N, torch.bfloat16, gated, True, False)
    x, w, bias, dy = given["x"], given["w"], given["bias"], given["dy"]
    saved = forward_kept(x, w, bias, "silu", gated)
    held = torch.full((1 << 28,), float("nan"), device=DEV).view(torch.uint8)
    *got, _ = backward(dy, x, w, bias, saved, "silu", gated, want, held)
    check_gradients(got, want, x, w, bias, dy, "silu", gated)
