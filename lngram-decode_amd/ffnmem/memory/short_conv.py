"""The short causal depthwise convolution on its own: bias, activation, dilation, a history of earlier
rows, ragged lengths, a backward pass, and the step for one new token of every sequence.

``DepthwiseCausalConv`` (the conv of the reference's memory layer, ``ffnmem/memory/lngram_v2.py:207-311``)
runs it for its bias and LayerNorm forms, ``SelectiveSSM`` as its token mixer.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from lngram_hip import ops

from .grad_mode import needs_grad

ACTIVATIONS = ("silu", None)


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, history, lengths, dilation: int, silu: bool):
        y, nxt = ops.short_conv(x, weight, bias, dilation, silu, history, lengths, want_history=True)
        ctx.save_for_backward(x, weight, bias, history, lengths)
        ctx.cfg = (dilation, silu)
        ctx.set_materialize_grads(False)
        return y, nxt

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnext):
        x, weight, bias, history, lengths = ctx.saved_tensors
        if dy is None:
            dy = x.new_zeros(1).expand(x.shape)
        dx, dw, db, dh = ops.short_conv_grad(dy, x, weight, bias, *ctx.cfg, history, lengths, dnext,
                                             ctx.needs_input_grad[:4])
        return dx, dw, db, dh, None, None, None


def _weight(weight: Tensor) -> Tensor:
    """``[C, K]`` from that or from ``nn.Conv1d``'s ``[C, 1, K]``."""
    return weight.squeeze(1) if weight.dim() == 3 and weight.shape[1] == 1 else weight


def _is_silu(activation: Optional[str]) -> bool:
    if activation not in ACTIVATIONS:
        raise ValueError(f"short conv activation must be one of {ACTIVATIONS}, got {activation!r}")
    return activation == "silu"


def short_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, dilation: int = 1,
               activation: Optional[str] = "silu", history: Optional[Tensor] = None,
               lengths: Optional[Tensor] = None, return_history: bool = False):
    """``act(bias + sum_j weight[:, j] * x[t - (K - 1 - j) * dilation])`` for x ``[B, T, C]`` (fp32, bf16 or
    fp16, channels contiguous or copied so), weight ``[C, K]`` or ``[C, 1, K]`` of 1 to 8 taps and bias
    ``[C]`` in x's type or fp32.

    ``history [B, (K - 1) * dilation, C]`` holds the rows before the first position (None: zeros).
    ``lengths [B]`` are the sequences' own tokens in a padded batch: positions behind them are not read,
    and give zeros.  ``return_history``: also the history of the tokens that follow each sequence's last own
    one.  Differentiable once, in reverse mode, in x, weight, bias and history."""
    w, silu = _weight(weight), _is_silu(activation)
    if needs_grad(x, w, bias, history):
        y, nxt = _ShortConv.apply(x, w, bias, history, lengths, int(dilation), silu)
        return (y, nxt) if return_history else y
    return ops.short_conv(x, w, bias, dilation, silu, history, lengths, return_history)


def short_conv_step(x: Tensor, history: Tensor, weight: Tensor, bias: Optional[Tensor] = None, dilation: int = 1,
                    activation: Optional[str] = "silu", out_history: Optional[Tensor] = None) -> Tensor:
    """:func:`short_conv` of one new token x ``[B, C]`` of every sequence.  ``history`` moves on by one row in
    place; with ``out_history`` the new one is written there and ``history`` stays (a step that may have to
    be taken back).  No gradient: call it under ``torch.no_grad()``."""
    if needs_grad(x, history, weight, bias):
        raise RuntimeError("short_conv_step has no backward pass; call it under torch.no_grad()")
    return ops.short_conv_step(x, history, _weight(weight), bias, dilation, _is_silu(activation), out_history)
