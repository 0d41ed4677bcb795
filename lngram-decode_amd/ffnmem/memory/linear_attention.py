"""Linear attention with a decay for each head: a matrix state per head where ``DiagonalSSM``
(``ffnmem/memory/ssm.py:22-55``) has a number and ``SelectiveSSM`` a few a channel.

    S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,      y[t] = scale S[t]^T q[t]

``linear_attention`` is the recurrence for prompts and training, ``linear_attention_step`` for one new token of
every sequence; ``LinearAttentionSSM`` makes the token router's SSM context (``router_input="embed2_ssm"``) from them.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from lngram_hip import ops

from .grad_mode import needs_grad
from .norm import GroupNorm, LayerNorm
from .selective import own_rows, project


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


class LinearAttentionSSM(nn.Module):
    """The token router's SSM context from a matrix state per head, where ``DiagonalSSM`` keeps a number a feature::

        x = LayerNorm(E[x[t]]);   q, k, v = W_qkv x;   g = log sigmoid(W_g x + b)
        S[t] = exp(g) S[t-1] + k v^T,   features = silu(GroupNorm(S[t]^T q / sqrt(key_dim)))

    with a group a head in the norm: heads of a long memory sum over more tokens than those of a short one.
    ``state_dim`` features from ``heads`` heads; ``kv_heads`` (None: ``heads``) of them keys and values of their own,
    shared by neighbours.  The decays of an input of zeros start between ``decay_min`` and ``decay_max``, their time
    constants spaced geometrically over the heads as ``DiagonalSSM``'s are over its channels
    (``ffnmem/memory/ssm.py:22-55``).

    ``forward`` takes whole sequences (differentiable), ``step`` one token of every sequence; both carry the same
    state ``[B, heads, key_dim, state_dim / heads]`` (fp32) and leave the one they are given as it was, so that
    taking tokens back is keeping an earlier one.  Weights in fp32 or bf16."""

    def __init__(self, d_model: int, state_dim: int = 256, heads: int = 4, key_dim: int = 64,
                 kv_heads: Optional[int] = None, eps: float = 1e-5, init_std: float = 0.02, decay_min: float = 0.5,
                 decay_max: float = 0.999):
        super().__init__()
        self.state_dim, self.heads, self.key_dim = int(state_dim), int(heads), int(key_dim)
        self.kv_heads = self.heads if kv_heads is None else int(kv_heads)
        if self.heads < 1 or self.state_dim % self.heads or not 1 <= self.state_dim // self.heads <= 128:
            raise ValueError(f"heads that divide state_dim into 1 to 128 values each, got {heads} of {state_dim}")
        if not 1 <= self.key_dim <= 128 or self.kv_heads < 1 or self.heads % self.kv_heads:
            raise ValueError("key_dim is 1 to 128, kv_heads divide the heads")
        if not 0.0 < decay_min <= decay_max < 1.0:
            raise ValueError("decays need 0 < decay_min <= decay_max < 1")
        self.value_dim = self.state_dim // self.heads
        self._widths = (self.heads * self.key_dim, self.kv_heads * self.key_dim, self.kv_heads * self.value_dim)
        self.norm = LayerNorm(d_model, eps)
        self.w_qkv = nn.Linear(d_model, sum(self._widths), bias=False)
        self.w_g = nn.Linear(d_model, self.heads, bias=False)
        for w in (self.w_qkv, self.w_g):
            nn.init.normal_(w.weight, mean=0.0, std=init_std)
        gone = torch.exp(torch.linspace(math.log(1 - decay_min), math.log(1 - decay_max), self.heads))
        self.decay_bias = nn.Parameter(torch.log1p(-gone) - torch.log(gone))
        self.out_norm = GroupNorm(self.heads, self.state_dim, eps, activation="silu")

    def empty_state(self, batch: int) -> Tensor:
        """The state before the first token."""
        return torch.zeros(batch, self.heads, self.key_dim, self.value_dim, dtype=torch.float32,
                           device=self.w_qkv.weight.device)

    def _inputs(self, emb: Tensor) -> tuple:
        x = self.norm(emb.to(self.w_qkv.weight.dtype))
        q, k, v = project(x, self.w_qkv).split(self._widths, dim=-1)
        g = nn.functional.logsigmoid(project(x, self.w_g).float() + self.decay_bias.float())
        return (q.unflatten(-1, (self.heads, self.key_dim)), k.unflatten(-1, (self.kv_heads, self.key_dim)),
                v.unflatten(-1, (self.kv_heads, self.value_dim)), g)

    def forward(self, emb: Tensor, state: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                return_state: bool = False):
        """Features ``[B, T, state_dim]`` of the embeddings ``[B, T, d]`` that follow ``state`` (None: the sequence
        start); with ``return_state`` also the state after each sequence's last own token.  ``lengths [B]``: the
        sequences' own tokens; what stands behind them has no part in features, state or gradients."""
        b, t = emb.shape[:2]
        out = linear_attention(*self._inputs(own_rows(emb, lengths)), state=state, lengths=lengths,
                               return_state=return_state)
        y, state = out if return_state else (out, None)
        y = self.out_norm(y.reshape(b * t, self.state_dim)).view(b, t, self.state_dim)
        if lengths is not None:                              # the norm's bias is no feature of no token
            y = y.masked_fill((torch.arange(t, device=y.device) >= lengths[:, None])[..., None], 0)
        return (y, state) if return_state else y

    @torch.no_grad()
    def step(self, state: Optional[Tensor], emb_t: Tensor) -> tuple:
        """``(features [B, state_dim], new state)`` of one token ``emb_t [B, d]`` of every sequence."""
        if state is None:
            state = self.empty_state(emb_t.shape[0])
        new = torch.empty_like(state)
        y = linear_attention_step(state, *self._inputs(emb_t), out_state=new)
        return self.out_norm(y.view(emb_t.shape[0], self.state_dim)), new
