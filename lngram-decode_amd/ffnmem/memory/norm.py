"""Layer norm with its backward pass (``nn.LayerNorm``, the LayerNorm choice of the reference's
``build_lngram_norm``, ``ffnmem/memory/lngram_v2.py:56-71``), and group norm of channels-last rows with an
activation behind it.

Statistics, sums and the weights' gradients are fp32; every output is rounded once.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from lngram_hip import ops

from .grad_mode import needs_grad


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> Tensor:
        y, mean, rstd = ops.layer_norm(x, weight, bias, eps, want_stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.w_dtype = next((t.dtype for t in (weight, bias) if t is not None), None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        x, weight, mean, rstd = ctx.saved_tensors
        return (*ops.layer_norm_grad(dy, x, weight, mean, rstd, ctx.needs_input_grad[:3], ctx.w_dtype), None)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of x (fp32, bf16 or fp16,
    any strides); weight and bias ``[d]`` in x's type or fp32, or None.  Differentiable once,
    in reverse mode."""
    if needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return ops.layer_norm(x, weight, bias, float(eps))


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float, silu: bool) -> Tensor:
        # what the backward pass can be spared is done here: it runs on autograd's own thread, whose host work is slow
        y, stats, ctx.plan, tensors = ops.group_norm_plan(x, groups, weight, bias, eps, silu, True)
        ctx.save_for_backward(*tensors, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        return (*ops.group_norm_back(ctx.plan, ctx.saved_tensors, dy, ctx.needs_input_grad), None, None, None)


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               activation: Optional[str] = None) -> Tensor:
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` of channels-last x ``[N, .., C]`` (fp32, bf16 or fp16):
    mean and variance of each of ``groups`` groups of neighbouring channels over all positions of a sample.  Tokens
    that are normed on their own are samples of one position, ``x [N, C]``.  weight and bias ``[C]`` in x's type or
    fp32, or None; ``activation`` None or "silu".  Differentiable once, in reverse mode."""
    if activation not in (None, "silu"):
        raise ValueError(f"group norm activation must be None or 'silu', got {activation!r}")
    if needs_grad(x, weight, bias):
        return _GroupNorm.apply(x, weight, bias, int(groups), float(eps), activation == "silu")
    return ops.group_norm(x, int(groups), weight, bias, float(eps), activation == "silu")


def rows_type(parameter: Optional[Tensor], rows: Tensor) -> Optional[Tensor]:
    """A parameter as the kernels take it beside ``rows``: as it is in the rows' type or fp32, else cast to the
    rows' type (as ``RMSNorm`` casts its weight)."""
    if parameter is None or parameter.dtype in (rows.dtype, torch.float32):
        return parameter
    return parameter.to(rows.dtype)


class LayerNorm(nn.Module):
    """``nn.LayerNorm(hidden_size, eps)``: parameters ``weight`` (ones) and ``bias`` (zeros)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        self.hidden_size = int(hidden_size)
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(hidden_size, device=device, dtype=dtype))

    def forward(self, hidden_states: Tensor) -> Tensor:
        if hidden_states.shape[-1] != self.hidden_size:
            raise ValueError(f"LayerNorm expects last dim {self.hidden_size}, got {hidden_states.shape[-1]}")
        return layer_norm(hidden_states, rows_type(self.weight, hidden_states), rows_type(self.bias, hidden_states),
                          self.eps)


class GroupNorm(nn.Module):
    """Group norm of channels-last rows, ``nn.GroupNorm(groups, channels, eps)``'s parameters ``weight`` (ones) and
    ``bias`` (zeros), with an activation behind it."""

    def __init__(self, groups: int, channels: int, eps: float = 1e-5, activation: Optional[str] = None, device=None,
                 dtype=None):
        super().__init__()
        if groups < 1 or channels % groups:
            raise ValueError(f"groups that divide the {channels} channels, got {groups}")
        if activation not in (None, "silu"):
            raise ValueError(f"group norm activation must be None or 'silu', got {activation!r}")
        self.groups, self.channels, self.eps, self.activation = int(groups), int(channels), float(eps), activation
        self.weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1] != self.channels:
            raise ValueError(f"GroupNorm expects last dim {self.channels}, got {x.shape[-1]}")
        return group_norm(x, self.groups, rows_type(self.weight, x), rows_type(self.bias, x), self.eps, self.activation)
