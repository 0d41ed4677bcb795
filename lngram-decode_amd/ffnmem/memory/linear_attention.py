"""Linear attention with a decay for each head: a matrix state per head where ``DiagonalSSM``
(``ffnmem/memory/ssm.py:22-55``) has a number and ``SelectiveSSM`` a few a channel.

    S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,      y[t] = scale S[t]^T q[t]

``linear_attention`` is the recurrence for prompts and training, ``linear_attention_step`` for one new token of
every sequence.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from lngram_hip import ops

from .grad_mode import needs_grad


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state, lengths, scale, want_state: bool):
        # what the backward pass can be spared is done here: it runs on autograd's own thread, whose host work is slow
        y, end, _, ctx.plan, tensors = ops.linear_attention_plan(q, k, v, decay, scale, state, lengths, want_state, True)
        ctx.save_for_backward(*tensors)
        ctx.set_materialize_grads(False)
        return y, end

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dend):
        tensors = ctx.saved_tensors
        if dy is None:
            _, q, _, v, decay, _, _ = tensors
            dy = q.new_zeros(1).expand(*q.shape[:2], decay.shape[-1], v.shape[-1])
        grads = ops.linear_attention_back(ctx.plan, tensors, dy, dend)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def _f32(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.dtype == torch.float32 else t.float()


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, scale: Optional[float] = None,
                     state: Optional[Tensor] = None, lengths: Optional[Tensor] = None, return_state: bool = False):
    """Linear attention over q ``[B, T, Hq, K]``, k ``[B, T, Hk, K]`` and v ``[B, T, Hv, V]``::

        S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,   y[t] = scale S[t]^T q[t]

    ``log_decay``: g, one a head ``[H]`` or one a token and head ``[B, T, H]``, in fp32 or converted to it (minus
    infinity clears the state; positive ones grow it).  The heads of q, k and v divide H: fewer are shared by
    neighbouring heads.  q, k and v in one type (fp32, bf16 or fp16; views whose last dimension is contiguous
    are read in place), 1 to 128 keys and values a head.  ``scale`` None: ``K ** -0.5``.  ``state [B, H, K, V]``:
    the state before the first token (None: zeros).  ``lengths [B]``: the sequences' own tokens in a padded
    batch; positions behind them are not read and give zeros.  Returns y ``[B, T, H, V]`` in q's type, with
    ``return_state`` also the state after each sequence's last own token (fp32).  States and sums are fp32.
    Differentiable once, in reverse mode, in everything but the lengths."""
    log_decay, state = _f32(log_decay), _f32(state)
    if needs_grad(q, k, v, log_decay, state):
        y, end = _LinearAttention.apply(q, k, v, log_decay, state, lengths, scale, bool(return_state))
    else:
        y, end, _ = ops.linear_attention(q, k, v, log_decay, scale, state, lengths, return_state)
    return (y, end) if return_state else y


def linear_attention_step(state: Tensor, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor,
                          scale: Optional[float] = None, out_state: Optional[Tensor] = None) -> Tensor:
    """:func:`linear_attention` of one new token of every sequence: q ``[B, Hq, K]``, k ``[B, Hk, K]``, v
    ``[B, Hv, V]``, log_decay ``[H]`` or ``[B, H]``; returns y ``[B, H, V]``.  ``state [B, H, K, V]`` (fp32,
    contiguous) moves on in place; with ``out_state`` the new one is written there and ``state`` stays (a step
    that may have to be taken back).  No gradient: call it under ``torch.no_grad()``."""
    if needs_grad(state, q, k, v, log_decay):
        raise RuntimeError("linear_attention_step has no backward pass; call it under torch.no_grad()")
    return ops.linear_attention_step(state, q, k, v, _f32(log_decay), scale, out_state)
