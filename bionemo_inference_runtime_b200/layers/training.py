"""Trainable layers: layer norm, dense and gated dense (with adapters) and dropout with gradients, and a transition made of them.

The inference layers fold their weights once and have no backward pass.  The functions here are differentiable (first
order, reverse mode) and read plain weights, so that a transition of a trunk can be fine-tuned and its weights handed back:
:class:`TrainableTransition` has the parameters and ``state_dict`` keys of
:class:`~bionemo_inference_runtime_b200.Transition` (``bionemo_ir/_torch/layers/transition.py:187-336`` of the reference,
which is forward only).  Instead of its weights, low-rank adapters beside them can be trained and many of them served in one
batch.  bf16 and fp16, any widths; layer norm and dropout also in fp32.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops
from .transition import _row_mask


def _refuse_capture(ctx, dy: torch.Tensor) -> None:
    """Refuses, by name, a captured backward pass whose gradients go to leaves that an eager graph holds on the default stream."""
    if dy.is_cuda and torch.cuda.is_current_stream_capturing():
        leaves = [f.variable for f, _ in ctx.next_functions if f is not None and f.name() == "torch::autograd::AccumulateGrad"]
        if ops._host.accumulated_elsewhere(leaves):
            raise RuntimeError("a backward pass is captured into a graph while an eager graph of the same leaves is alive, whose gradients are "
                               "accumulated on the default stream: release that graph first")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ops.layer_norm(x, weight, bias, eps, want_stats=True)
        ctx.save_for_backward(x, stats, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture(ctx, dy)
        x, stats, weight = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        dx, dweight, dbias = ops.layer_norm_backward(dy, x, stats, weight, want_dx=wanted[0], want_dweight=wanted[1],
                                                     want_dbias=wanted[2])
        return dx, dweight, dbias, None


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        keep = any(ctx.needs_input_grad[:3])  # the gradient of the residual is dy
        y = ops.dense(x, weight, bias, activation=activation, residual=residual, want_saved=keep)
        y, saved = y if keep else (y, None)
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture(ctx, dy)
        x, weight, bias, saved = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        grads = (None, None, None)
        if any(wanted[:3]):
            grads = ops.dense_backward(dy, x, weight, bias, activation=ctx.activation, saved=saved, want_dx=wanted[0],
                                       want_dweight=wanted[1], want_dbias=wanted[2])
        return (*grads, dy if wanted[3] else None, None)


class _GatedDense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation):
        y, saved = ops.gated_dense(x, weight, bias, activation=activation, want_saved=True)
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture(ctx, dy)
        x, weight, bias, saved = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        grads = ops.gated_dense_backward(dy, x, weight, bias, activation=ctx.activation, saved=saved, want_dx=wanted[0],
                                         want_dweight=wanted[1], want_dbias=wanted[2])
        return (*grads, None)


class _AdapterDense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, down, up, residual, index, scale, activation, gated):
        forward, more = (ops.adapter_gated_dense, {}) if gated else (ops.adapter_dense, {"residual": residual})
        keep = any(ctx.needs_input_grad[:5])
        y = forward(x, weight, bias, down, up, index, scale, activation=activation, want_saved=keep, **more)
        y, saved = y if keep else (y, (None, None))
        at = scale if isinstance(scale, torch.Tensor) else None
        ctx.save_for_backward(x, weight, bias, down, up, index, at, *saved)
        ctx.scale = None if at is not None else scale
        ctx.activation, ctx.gated = activation, gated
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture(ctx, dy)
        x, weight, bias, down, up, index, scale, *saved = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        grads = (None,) * 5
        if any(wanted[:5]):
            backward = ops.adapter_gated_dense_backward if ctx.gated else ops.adapter_dense_backward
            grads = backward(dy, x, weight, bias, down, up, index, ctx.scale if scale is None else scale, activation=ctx.activation, saved=tuple(saved),
                             want_dx=wanted[0], want_dweight=wanted[1], want_dbias=wanted[2], want_ddown=wanted[3], want_dup=wanted[4])
        return (*grads, dy if wanted[5] else None, None, None, None, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, sequence, shared):
        if isinstance(seed, torch.Tensor):
            seed = seed.clone()  # a later step's seed may be written to the tensor before this step's backward pass
        ctx.given = (p, seed, sequence)
        ctx.shared = shared
        return ops.dropout(x, p, seed, sequence, residual=residual, shared=shared)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture(ctx, dy)
        dx = ops.dropout_backward(dy, *ctx.given, shared=ctx.shared) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def _needs_grad(*tensors: torch.Tensor | None) -> bool:
    # A tensor with a tangent need not require a gradient: its result would silently have no tangent.  (Outside of a level there
    # are none; asking each tensor costs 0.4 us.)
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the trainable layers have no forward-mode derivatives")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Differentiable :func:`ops.layer_norm <bionemo_inference_runtime_b200.ops.layer_norm>`."""
    return _LayerNorm.apply(x, weight, bias, eps) if _needs_grad(x, weight, bias) else ops.layer_norm(x, weight, bias, eps)


def dense(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
          residual: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable :func:`ops.dense <bionemo_inference_runtime_b200.ops.dense>`:
    ``activation(x @ weight.T + bias) + residual``."""
    if _needs_grad(x, weight, bias, residual):
        return _Dense.apply(x, weight, bias, residual, activation)
    return ops.dense(x, weight, bias, activation=activation, residual=residual)


def gated_dense(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                activation: str = "silu") -> torch.Tensor:
    """Differentiable :func:`ops.gated_dense <bionemo_inference_runtime_b200.ops.gated_dense>`:
    ``value * activation(gate)``, ``[value | gate] = x @ weight.T + bias``."""
    if _needs_grad(x, weight, bias):
        return _GatedDense.apply(x, weight, bias, activation)
    return ops.gated_dense(x, weight, bias, activation=activation)


def _adapter_dense(x, weight, bias, down, up, residual, index, scale, activation, gated):
    if isinstance(scale, torch.Tensor) and _needs_grad(scale):
        raise NotImplementedError("the scale of adapters has no gradient")
    if not _needs_grad(x, weight, bias, down, up, residual):
        if gated:
            return ops.adapter_gated_dense(x, weight, bias, down, up, index, scale, activation=activation)
        return ops.adapter_dense(x, weight, bias, down, up, index, scale, activation=activation, residual=residual)
    return _AdapterDense.apply(x, weight, bias, down, up, residual, index, scale, activation, gated)


def adapter_dense(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, down: torch.Tensor, up: torch.Tensor,
                  index: torch.Tensor | None = None, scale: float | torch.Tensor = 1.0, *, activation: str = "none",
                  residual: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable :func:`ops.adapter_dense <bionemo_inference_runtime_b200.ops.adapter_dense>`:
    ``activation(x @ weight.T + bias + scale[g] * (x @ down[g].T) @ up[g].T) + residual``."""
    return _adapter_dense(x, weight, bias, down, up, residual, index, scale, activation, False)


def adapter_gated_dense(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, down: torch.Tensor, up: torch.Tensor,
                        index: torch.Tensor | None = None, scale: float | torch.Tensor = 1.0, *,
                        activation: str = "silu") -> torch.Tensor:
    """Differentiable :func:`ops.adapter_gated_dense <bionemo_inference_runtime_b200.ops.adapter_gated_dense>`:
    ``value * activation(gate)``, both with their part of the adapter."""
    return _adapter_dense(x, weight, bias, down, up, None, index, scale, activation, True)


def dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, sequence: int = 0, *, residual: torch.Tensor | None = None,
            shared: int | None = None) -> torch.Tensor:
    """Differentiable :func:`ops.dropout <bionemo_inference_runtime_b200.ops.dropout>`: ``residual + keep * x / (1 - p)``."""
    if _needs_grad(x, residual):
        return _Dropout.apply(x, residual, p, seed, sequence, shared)
    return ops.dropout(x, p, seed, sequence, residual=residual, shared=shared)


class _Weight(nn.Module):
    """``weight[out, in]`` drawn like that of ``torch.nn.Linear``."""

    def __init__(self, in_features: int, out_features: int, dtype: torch.dtype, device):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(out_features, in_features, dtype=dtype, device=device))
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))


class _Adapters(nn.Module):
    """``down[adapters, rank, in]`` drawn like a weight, ``up[adapters, out, rank]`` zero: an adapter that changes nothing yet."""

    def __init__(self, adapters: int, rank: int, in_features: int, out_features: int, dtype: torch.dtype, device):
        super().__init__()
        self.down = nn.Parameter(torch.empty(adapters, rank, in_features, dtype=dtype, device=device))
        self.up = nn.Parameter(torch.zeros(adapters, out_features, rank, dtype=dtype, device=device))
        for one in self.down:
            nn.init.kaiming_uniform_(one, a=math.sqrt(5))


class TrainableTransition(nn.Module):
    """``[x +] [mask *] fc3(silu(gate) * value)``, ``[value | gate] = fused_fc2_fc1(norm(x))``, with gradients for ``x`` and
    all parameters.

    Constructor arguments, ``forward`` and ``state_dict`` keys are those of ``Transition`` (without the in-place form), the
    widths are free; ``Transition(...).load_state_dict(trained.state_dict())`` serves what was trained.

    With ``adapter_rank`` both dense layers have ``adapters`` low-rank adapters beside their weights
    (``fused_fc2_fc1_adapters`` and ``fc3_adapters``), multiplied by ``adapter_scale``; the other parameters begin frozen.
    ``forward`` then takes the ``index`` of :func:`adapter_dense`, and :meth:`merged_state_dict` gives the weights with one adapter
    added to them, as ``Transition`` loads them.  In training mode the update is dropped with probability ``dropout`` before it joins
    the residual, by one draw for all entries along the axis ``dropout_shared`` of ``x``.
    """

    def __init__(self, dim: int, hidden: int, out_dim: int | None = None, eps: float = 1e-5,
                 dtype: torch.dtype = torch.bfloat16, normalize: bool = True, device=None, *, dropout: float = 0.0,
                 dropout_shared: int | None = None, adapter_rank: int = 0, adapters: int = 1, adapter_scale: float = 1.0):
        super().__init__()
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the dense layers compute in bfloat16 or float16, got {dtype}")
        if not 0 <= dropout <= 1:
            raise ValueError(f"dropout must lie between 0 and 1, got {dropout}")
        if adapter_rank < 0 or adapter_rank > 256 or adapters < 1:
            raise ValueError(f"adapters need a rank of 1 to 256, got {adapters} of rank {adapter_rank}")
        self.dim, self.hidden, self.out_dim = dim, hidden, dim if out_dim is None else out_dim
        self.dtype = dtype
        device = device if device is not None else "cuda" if torch.cuda.is_available() else "cpu"
        self.norm = nn.LayerNorm(dim, eps=eps, dtype=dtype, device=device) if normalize else None
        self.fused_fc2_fc1 = _Weight(dim, 2 * hidden, dtype, device)
        self.fc3 = _Weight(hidden, self.out_dim, dtype, device)
        self.dropout, self.dropout_shared, self.adapter_scale = dropout, dropout_shared, adapter_scale
        self.fused_fc2_fc1_adapters = self.fc3_adapters = None
        if adapter_rank:
            self.requires_grad_(False)
            self.fused_fc2_fc1_adapters = _Adapters(adapters, adapter_rank, dim, 2 * hidden, dtype, device)
            self.fc3_adapters = _Adapters(adapters, adapter_rank, hidden, self.out_dim, dtype, device)

    def merged_state_dict(self, adapter: int = 0) -> dict[str, torch.Tensor]:
        """The ``state_dict`` of a ``Transition`` that computes what this one does for rows of an adapter (its products are rounded
        to the weights' dtype)."""
        state = {k: v for k, v in self.state_dict().items() if "_adapters." not in k}
        if self.fc3_adapters is None:
            return state
        if not 0 <= adapter < self.fc3_adapters.down.shape[0]:
            raise ValueError(f"there is no adapter {adapter} of {self.fc3_adapters.down.shape[0]}")
        for name, adapters in (("fused_fc2_fc1", self.fused_fc2_fc1_adapters), ("fc3", self.fc3_adapters)):
            weight = state[f"{name}.weight"]
            added = adapters.up[adapter].detach().double() @ adapters.down[adapter].detach().double()
            state[f"{name}.weight"] = (weight.double() + self.adapter_scale * added).to(weight.dtype)
        return state

    def _gated(self, x, index):
        if self.fused_fc2_fc1_adapters is None:
            return gated_dense(x, self.fused_fc2_fc1.weight)
        a = self.fused_fc2_fc1_adapters
        return adapter_gated_dense(x, self.fused_fc2_fc1.weight, None, a.down, a.up, index, self.adapter_scale)

    def _out(self, x, index, residual):
        if self.fc3_adapters is None:
            return dense(x, self.fc3.weight, residual=residual)
        a = self.fc3_adapters
        return adapter_dense(x, self.fc3.weight, None, a.down, a.up, index, self.adapter_scale, residual=residual)

    def forward(self, x: torch.Tensor, mask: torch.Tensor | None = None, *, residual: bool = False,
                index: torch.Tensor | None = None, seed: int | torch.Tensor | None = None, sequence: int = 0) -> torch.Tensor:
        """``seed`` and ``sequence`` are those of :func:`dropout`; without a seed one is drawn from PyTorch's CPU generator (a step that
        is captured into a graph needs one, on the device if it is to be another one at each replay)."""
        if residual and self.out_dim != self.dim:
            raise ValueError(f"a residual needs out_dim == dim, got {self.out_dim} and {self.dim}")
        if index is not None and self.fc3_adapters is None:
            raise ValueError("an index needs adapters (adapter_rank)")
        normed = x if self.norm is None else layer_norm(x, self.norm.weight, self.norm.bias, self.norm.eps)
        update = self._gated(normed, index)
        drops = self.training and self.dropout > 0
        if mask is None and not drops:
            return self._out(update, index, x if residual else None)
        update = self._out(update, index, None)
        if mask is not None:
            update = update * _row_mask(x, mask).unsqueeze(-1).to(x.dtype)
        if drops:
            if seed is None:
                if x.is_cuda and torch.cuda.is_current_stream_capturing():
                    raise ValueError("a captured step needs a seed: one drawn now would drop the same elements at every replay")
                seed = int(torch.randint(1 << 62, ()))
            return dropout(update, self.dropout, seed, sequence, residual=x if residual else None, shared=self.dropout_shared)
        return x + update if residual else update
