"""Selective state space over token embeddings: the SSM context of the token router
(``router_input="embed2_ssm"``) with step sizes, inputs and outputs that each token chooses, where
``DiagonalSSM`` (``ffnmem/memory/ssm.py:22-55``) has one decay a channel for all tokens.

    x, z  = W_in LayerNorm(E[x[t]])
    u     = silu(short causal conv of x)
    dt, B, C = W_x u;   s = softplus(W_dt dt + dt_bias)
    h[t]  = exp(s A) h[t-1] + s u B,    A = -exp(A_log)
    y[t]  = (C h[t] + D u) silu(z)

``selective_scan`` is the recurrence for prompts and training, ``selective_step`` for one new token of every
sequence.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from lngram_hip import ops

from .grad_mode import needs_grad
from .norm import LayerNorm
from .short_conv import short_conv, short_conv_step


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus: bool, want_state: bool):
        y, end, ckpt = ops.selective_scan(u, dt, A, B, C, D, z, dt_bias, softplus, state, lengths, want_state, True)
        ctx.save_for_backward(ckpt, u, dt, A, B, C, D, z, dt_bias, state, lengths)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, end

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dend):
        ckpt, u, dt, A, B, C, D, z, dt_bias, state, lengths = ctx.saved_tensors
        if dy is None:
            dy = u.new_zeros(1).expand(u.shape)
        g = ops.selective_scan_grad(dy, dend, ckpt, u, dt, A, B, C, D, z, dt_bias, ctx.softplus, state, lengths)
        names = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")
        return (*(g.get(k) if need else None for k, need in zip(names, ctx.needs_input_grad)), None, None, None)


def _f32(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.dtype == torch.float32 else t.float()


def selective_scan(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor] = None,
                   z: Optional[Tensor] = None, dt_bias: Optional[Tensor] = None, dt_softplus: bool = False,
                   state: Optional[Tensor] = None, lengths: Optional[Tensor] = None, return_state: bool = False):
    """The selective scan of u ``[B, T, C]``::

        s = softplus(dt + dt_bias)  (dt_softplus) or dt + dt_bias
        h[t] = exp(s A) h[t-1] + s u B[t],   y[t] = (C[t] . h[t] + D u) * silu(z)

    u, dt, z ``[B, T, C]`` and B, C ``[B, T, N]`` or ``[B, T, G, N]`` (G groups of neighbouring channels) in
    one type (fp32, bf16 or fp16; views whose last dimension is contiguous are read in place); A ``[C, N]``,
    D ``[C]``, dt_bias ``[C]`` and ``state [B, C, N]`` (the state before the first token, None: zeros) in
    fp32 or converted to it; 1 to 256 states.  ``lengths [B]``: the sequences' own tokens in a padded batch;
    positions behind them are not read and give zeros.  Returns y ``[B, T, C]`` in u's type, with
    ``return_state`` also the state after each sequence's last own token (fp32).  States and sums are fp32.
    Differentiable once, in reverse mode, in everything but the lengths."""
    A, D, dt_bias, state = _f32(A), _f32(D), _f32(dt_bias), _f32(state)
    if needs_grad(u, dt, A, B, C, D, z, dt_bias, state):
        y, end = _SelectiveScan.apply(u, dt, A, B, C, D, z, dt_bias, state, lengths, bool(dt_softplus),
                                      bool(return_state))
    else:
        y, end, _ = ops.selective_scan(u, dt, A, B, C, D, z, dt_bias, dt_softplus, state, lengths, return_state)
    return (y, end) if return_state else y


def selective_step(state: Tensor, u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor] = None,
                   z: Optional[Tensor] = None, dt_bias: Optional[Tensor] = None, dt_softplus: bool = False,
                   out_state: Optional[Tensor] = None) -> Tensor:
    """:func:`selective_scan` of one new token of every sequence: u, dt, z ``[B, C]``, B, C ``[B, N]`` or
    ``[B, G, N]``; returns y ``[B, C]``.  ``state [B, C, N]`` (fp32, contiguous) moves on in place; with
    ``out_state`` the new one is written there and ``state`` stays (a step that may have to be taken back).
    No gradient: call it under ``torch.no_grad()``."""
    if needs_grad(state, u, dt, A, B, C, D, z, dt_bias):
        raise RuntimeError("selective_step has no backward pass; call it under torch.no_grad()")
    return ops.selective_step(state, u, dt, _f32(A), B, C, _f32(D), z, _f32(dt_bias), dt_softplus, out_state)


class _Linear(torch.autograd.Function):
    """``x . w^T`` on ``lng_linear``; its gradients are two plain matrix products."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return ops.linear(x, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        d2, x2 = dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1])
        return (torch.mm(d2, w).view(x.shape) if ctx.needs_input_grad[0] else None,
                torch.mm(d2.t(), x2) if ctx.needs_input_grad[1] else None)


def project(x: Tensor, w: nn.Linear) -> Tensor:
    """``x . w^T``, differentiable; rows of a width that the bf16 product does not read are padded."""
    weight, odd = w.weight, -x.shape[-1] % 8
    if odd and x.dtype == torch.bfloat16:                # it reads 16 bytes at a time
        x, weight = nn.functional.pad(x, (0, odd)), nn.functional.pad(weight, (0, odd))
    if needs_grad(x, weight):
        return _Linear.apply(x, weight)
    return ops.linear(x, weight)


def own_rows(emb: Tensor, lengths: Optional[Tensor]) -> Tensor:
    """A training batch with zeros behind its sequences: the gradients of norms and products sum over every row, those
    behind a sequence's end with a factor of zero, and a NaN there would come through."""
    if lengths is None or lengths.shape != emb.shape[:1] or not torch.is_grad_enabled():
        return emb
    behind = torch.arange(emb.shape[1], device=emb.device) >= lengths[:, None]
    return emb.masked_fill(behind[..., None], 0)


class SelectiveSSM(nn.Module):
    """Selective SSM whose output is the token router's SSM context: ``state_dim`` features a token, as
    ``DiagonalSSM``'s, from ``d_state`` states a feature.

    ``forward`` takes whole sequences (differentiable), ``step`` one token of every sequence; both carry the
    same state, ``(conv history [B, K - 1, state_dim], scan state [B, state_dim, d_state])``, and leave the
    one they are given as it was, so that taking tokens back is keeping an earlier one.  Weights in fp32 or
    bf16 (a product's rows that are no multiple of 8 values wide are padded there)."""

    def __init__(self, d_model: int, state_dim: int = 256, d_state: int = 16, conv_kernel: int = 4,
                 dt_rank: Optional[int] = None, eps: float = 1e-5, init_std: float = 0.02, dt_min: float = 1e-3,
                 dt_max: float = 1e-1):
        super().__init__()
        if not 0.0 < dt_min <= dt_max:
            raise ValueError("step sizes need 0 < dt_min <= dt_max")
        if not 1 <= int(conv_kernel) <= 8 or not 1 <= int(d_state) <= 256:
            raise ValueError("conv_kernel is 1 to 8 taps, d_state 1 to 256 states")
        self.state_dim, self.d_state, self.conv_kernel = int(state_dim), int(d_state), int(conv_kernel)
        self.dt_rank = max(1, math.ceil(d_model / 16)) if dt_rank is None else int(dt_rank)
        n = self.state_dim
        self.norm = LayerNorm(d_model, eps)
        self.w_in = nn.Linear(d_model, 2 * n, bias=False)
        self.conv = nn.Conv1d(n, n, self.conv_kernel, groups=n, bias=True)
        self.w_x = nn.Linear(n, self.dt_rank + 2 * self.d_state, bias=False)
        self.w_dt = nn.Linear(self.dt_rank, n, bias=False)
        for w in (self.w_in, self.w_x):
            nn.init.normal_(w.weight, mean=0.0, std=init_std)
        nn.init.uniform_(self.w_dt.weight, -self.dt_rank ** -0.5, self.dt_rank ** -0.5)
        # step sizes spread over [dt_min, dt_max] geometrically, decay rates -1 .. -d_state
        step = torch.exp(torch.rand(n) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, self.d_state + 1, dtype=torch.float32)).repeat(n, 1))
        self.D = nn.Parameter(torch.ones(n))

    def empty_state(self, batch: int) -> tuple:
        """The state before the first token."""
        w = self.w_in.weight
        return (w.new_zeros(batch, self.conv_kernel - 1, self.state_dim),
                torch.zeros(batch, self.state_dim, self.d_state, dtype=torch.float32, device=w.device))

    _linear = staticmethod(project)

    def _inputs(self, emb: Tensor) -> tuple:
        return self._linear(self.norm(emb.to(self.w_in.weight.dtype)), self.w_in).chunk(2, dim=-1)

    def _selection(self, u: Tensor) -> tuple:
        low, bm, cm = self._linear(u, self.w_x).split((self.dt_rank, self.d_state, self.d_state), dim=-1)
        return self._linear(low, self.w_dt), bm, cm

    def forward(self, emb: Tensor, state: Optional[tuple] = None, lengths: Optional[Tensor] = None,
                return_state: bool = False):
        """Features ``[B, T, state_dim]`` of the embeddings ``[B, T, d]`` that follow ``state`` (None: the
        sequence start); with ``return_state`` also the state after each sequence's last own token.  ``lengths
        [B]``: the sequences' own tokens; what stands behind them has no part in features, state or gradients."""
        hist, scan = (None, None) if state is None else state
        x, z = self._inputs(own_rows(emb, lengths))
        u, hist = short_conv(x, self.conv.weight, self.conv.bias, history=hist, lengths=lengths, return_history=True)
        dt, bm, cm = self._selection(u)
        out = selective_scan(u, dt, -torch.exp(self.A_log.float()), bm, cm, D=self.D, z=z, dt_bias=self.dt_bias,
                             dt_softplus=True, state=scan, lengths=lengths, return_state=return_state)
        return (out[0], (hist, out[1])) if return_state else out

    @torch.no_grad()
    def step(self, state: Optional[tuple], emb_t: Tensor) -> tuple:
        """``(features [B, state_dim], new state)`` of one token ``emb_t [B, d]`` of every sequence."""
        hist, scan = self.empty_state(emb_t.shape[0]) if state is None else state
        new_hist, new_scan = torch.empty_like(hist), torch.empty_like(scan)
        x, z = self._inputs(emb_t)
        u = short_conv_step(x, hist, self.conv.weight, self.conv.bias, out_history=new_hist)
        dt, bm, cm = self._selection(u)
        y = selective_step(scan, u, dt, -torch.exp(self.A_log.float()), bm, cm, D=self.D, z=z, dt_bias=self.dt_bias,
                           dt_softplus=True, out_state=new_scan)
        return y, (new_hist, new_scan)
