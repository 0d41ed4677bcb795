"""Linear attention with a decay for each head, and group norm, in 64 bits (torch, CPU).

Each function gives the operator's outputs and, with ``dy``, its gradients by the formulas; with ``mag`` the
same sums over absolute values: the scale that a rounding error of an fp32 evaluation is proportional to.
"""

from __future__ import annotations

import torch
from torch import Tensor

FLUSH = 2.0 ** -102  # 2^24 times the smallest normal fp32 number: what an exponential below it is off by, in mag


def _heads(x: Tensor, h: int) -> Tensor:
    """Heads shared by neighbours repeated: [.., heads, width] -> [.., H, width]."""
    return x.repeat_interleave(h // x.shape[-2], -2)


def _shared(x: Tensor, heads: int) -> Tensor:
    return x.unflatten(-2, (heads, x.shape[-2] // heads)).sum(-2)


def _states(k, v, g, state, live, mag) -> list:
    """The states before the first token and after each one."""
    b, t = k.shape[:2]
    out = [k.new_zeros(b, k.shape[2], k.shape[3], v.shape[3]) if state is None else (state.abs() if mag else state)]
    for i in range(t):
        e = torch.exp(g[:, i])[..., None, None] + (FLUSH if mag else 0)
        s = e * out[-1] + k[:, i, :, :, None] * v[:, i, :, None]
        out.append(torch.where(live[:, i, None, None, None], s, out[-1]))
    return out


def _prepare(q, k, v, g, lengths, mag):
    b, t = q.shape[:2]
    h = g.shape[-1]
    q, k, v = (_heads(x.abs() if mag else x, h) for x in (q, k, v))
    own = torch.full((b,), t) if lengths is None else lengths.clamp(0, t).to("cpu").long()
    live = torch.arange(t)[None] < own[:, None]
    return q, k, v, g.expand(b, t, h), live


def linear_attention(q, k, v, g, scale, state=None, lengths=None, mag=False) -> tuple:
    """``(y, final state)``, token by token."""
    q, k, v, g, live = _prepare(q, k, v, g, lengths, mag)
    s = _states(k, v, g, state, live, mag)
    y = torch.stack([(q[:, i, :, :, None] * s[i + 1]).sum(2) * scale for i in range(q.shape[1])], 1) \
        if q.shape[1] else v.new_zeros(v.shape)
    return torch.where(live[..., None, None], y, 0.0), s[-1]


def linear_attention_grad(dy, dend, q, k, v, g, scale, state=None, lengths=None, mag=False, chunk=64) -> dict:
    """Gradients by their inputs' names.  ``mag`` of a decay's gradient: a chunk's pairs and states that an
    evaluation in chunks of up to ``chunk`` tokens adds up before some of them cancel."""
    hq, hk, hv = (x.shape[2] for x in (q, k, v))
    heads_g = g.dim() == 1
    q, k, v, g, live = _prepare(q, k, v, g, lengths, mag)
    if mag:
        dy, dend = dy.abs(), None if dend is None else dend.abs()
    dy = torch.where(live[..., None, None], dy, 0.0)
    b, t, h, _ = q.shape
    s = _states(k, v, g, state, live, mag)
    r = torch.zeros_like(s[0]) if dend is None else dend.clone()
    dq, dk, dv, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), q.new_zeros(b, t, h)
    for i in range(t - 1, -1, -1):
        on = live[:, i, None, None, None]
        rr = r + scale * q[:, i, :, :, None] * dy[:, i, :, None]
        dq[:, i] = scale * (s[i + 1] * dy[:, i, :, None]).sum(-1)
        dk[:, i] = (rr * v[:, i, :, None]).sum(-1)
        dv[:, i] = (rr * k[:, i, :, :, None]).sum(2)
        e = torch.exp(g[:, i])[..., None, None] + (FLUSH if mag else 0)
        dg[:, i] = (e * rr * s[i]).sum((-2, -1))
        r = torch.where(on, e * rr, r)
    for x in (dq, dk, dv):
        x[~live] = 0
    dg[~live] = 0
    if mag:                                          # what is added and taken away again within a chunk
        near = (q * dq).sum(-1) + (k * dk).sum(-1)
        acc = torch.cat((near.new_zeros(b, chunk, h), near, near.new_zeros(b, chunk, h)), 1).cumsum(1)
        dg = dg + acc[:, 2 * chunk - 1:2 * chunk - 1 + t] - acc[:, chunk - 1:chunk - 1 + t]    # t .. t + chunk - 1
        dg = dg + acc[:, chunk:chunk + t] - acc[:, :t]                                        # t - chunk + 1 .. t
    return dict(q=_shared(dq, hq), k=_shared(dk, hk), v=_shared(dv, hv), decay=dg.sum((0, 1)) if heads_g else dg, state=r)


# ----------------------------------------------------------------------------- group norm
def _rows(x: Tensor, groups: int) -> Tensor:
    """[N, .., C] -> [N, groups, positions, C / groups]."""
    n, c = x.shape[0], x.shape[-1]
    return x.reshape(n, x.numel() // max(n * c, 1) if n else 0, groups, c // groups).transpose(1, 2)


def _unrows(r: Tensor, shape) -> Tensor:
    return r.transpose(1, 2).reshape(shape)


def _sigmoid_parts(z: Tensor) -> tuple:
    s = torch.sigmoid(z)
    return s, s * (1 + z * (1 - s))


def group_norm(x: Tensor, groups: int, w, b, eps: float, silu: bool, mag=False) -> Tensor:
    r = _rows(x, groups)
    cg = r.shape[-1]
    mean = r.mean((2, 3), keepdim=True)
    xc = r - mean
    rstd = 1 / torch.sqrt((xc * xc).mean((2, 3), keepdim=True) + eps)
    wg = r.new_ones(groups, 1, cg) if w is None else w.view(groups, 1, cg)
    bg = r.new_zeros(groups, 1, cg) if b is None else b.view(groups, 1, cg)
    z = xc * rstd * wg + bg
    if mag:       # the mean's error moves a value by rstd * mean|x|
        m = wg.abs() * (xc.abs() * rstd + rstd * r.abs().mean((2, 3), keepdim=True)) + bg.abs()
        return _unrows(m * _sigmoid_parts(z)[1].abs().clamp_min(0.1) + (z * torch.sigmoid(z)).abs() * (1 + z.abs())
                       if silu else m, x.shape)
    return _unrows(z * torch.sigmoid(z) if silu else z, x.shape)


def group_norm_grad(dy: Tensor, x: Tensor, groups: int, w, b, eps: float, silu: bool, mag=False) -> tuple:
    """``(dx, dw, db)``."""
    r, d = _rows(x, groups), _rows(dy, groups)
    cg = r.shape[-1]
    mean = r.mean((2, 3), keepdim=True)
    xc = r - mean
    rstd = 1 / torch.sqrt((xc * xc).mean((2, 3), keepdim=True) + eps)
    wg = r.new_ones(groups, 1, cg) if w is None else w.view(groups, 1, cg)
    bg = r.new_zeros(groups, 1, cg) if b is None else b.view(groups, 1, cg)
    xn = xc * rstd
    z = xn * wg + bg
    if mag:
        # |xn| with the reach of the mean's error; the slope with that of z's error (its own slope is below 0.5)
        xn = xc.abs() * rstd + rstd * r.abs().mean((2, 3), keepdim=True)
        dz = d.abs() * (1.1 + 0.5 * (xn * wg.abs() + bg.abs()) if silu else 1.0)
        h = dz * wg.abs()
        dx = rstd * (h + h.mean((2, 3), keepdim=True) + xn * (h * xn).mean((2, 3), keepdim=True))
    else:
        dz = d * (_sigmoid_parts(z)[1] if silu else 1.0)
        h = dz * wg
        dx = rstd * (h - h.mean((2, 3), keepdim=True) - xn * (h * xn).mean((2, 3), keepdim=True))
    cols = [v.sum((0, 2)).reshape(-1) for v in (dz * xn, dz)]
    return _unrows(dx, x.shape), cols[0], cols[1]
