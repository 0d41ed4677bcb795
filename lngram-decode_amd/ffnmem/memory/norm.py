"""Layer norm with its backward pass (``nn.LayerNorm``, the LayerNorm choice of the reference's
``build_lngram_norm``, ``ffnmem/memory/lngram_v2.py:56-71``).

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
