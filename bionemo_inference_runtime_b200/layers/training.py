"""Trainable layers: layer norm, dense and gated dense with gradients, and a transition made of them.

The inference layers fold their weights once and have no backward pass.  The functions here are differentiable (first
order, reverse mode) and read plain weights, so that a transition of a trunk can be fine-tuned and its weights handed back:
:class:`TrainableTransition` has the parameters and ``state_dict`` keys of
:class:`~bionemo_inference_runtime_b200.Transition` (``bionemo_ir/_torch/layers/transition.py:187-336`` of the reference,
which is forward only).  bf16 and fp16, any widths; layer norm also in fp32.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops
from .transition import _row_mask


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ops.layer_norm(x, weight, bias, eps, want_stats=True)
        ctx.save_for_backward(x, stats, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
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
        x, weight, bias, saved = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        grads = ops.gated_dense_backward(dy, x, weight, bias, activation=ctx.activation, saved=saved, want_dx=wanted[0],
                                         want_dweight=wanted[1], want_dbias=wanted[2])
        return (*grads, None)


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


class _Weight(nn.Module):
    """``weight[out, in]`` drawn like that of ``torch.nn.Linear``."""

    def __init__(self, in_features: int, out_features: int, dtype: torch.dtype, device):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(out_features, in_features, dtype=dtype, device=device))
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))


class TrainableTransition(nn.Module):
    """``[x +] [mask *] fc3(silu(gate) * value)``, ``[value | gate] = fused_fc2_fc1(norm(x))``, with gradients for ``x`` and
    all parameters.

    Constructor arguments, ``forward`` and ``state_dict`` keys are those of ``Transition`` (without the in-place form), the
    widths are free; ``Transition(...).load_state_dict(trained.state_dict())`` serves what was trained.
    """

    def __init__(self, dim: int, hidden: int, out_dim: int | None = None, eps: float = 1e-5,
                 dtype: torch.dtype = torch.bfloat16, normalize: bool = True, device=None):
        super().__init__()
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the dense layers compute in bfloat16 or float16, got {dtype}")
        self.dim, self.hidden, self.out_dim = dim, hidden, dim if out_dim is None else out_dim
        self.dtype = dtype
        device = device if device is not None else "cuda" if torch.cuda.is_available() else "cpu"
        self.norm = nn.LayerNorm(dim, eps=eps, dtype=dtype, device=device) if normalize else None
        self.fused_fc2_fc1 = _Weight(dim, 2 * hidden, dtype, device)
        self.fc3 = _Weight(hidden, self.out_dim, dtype, device)

    def forward(self, x: torch.Tensor, mask: torch.Tensor | None = None, *, residual: bool = False) -> torch.Tensor:
        if residual and self.out_dim != self.dim:
            raise ValueError(f"a residual needs out_dim == dim, got {self.out_dim} and {self.dim}")
        normed = x if self.norm is None else layer_norm(x, self.norm.weight, self.norm.bias, self.norm.eps)
        update = gated_dense(normed, self.fused_fc2_fc1.weight)
        if mask is None:
            return dense(update, self.fc3.weight, residual=x if residual else None)
        update = dense(update, self.fc3.weight) * _row_mask(x, mask).unsqueeze(-1).to(x.dtype)
        return x + update if residual else update
