"""Layer norm, the short causal convolution and the selective state space scan in 64 bits (torch, CPU).

Each function gives the operator's outputs and, with ``dy``, its gradients by the formulas; ``mag``
companions evaluate the same sums over absolute values: the scale that a rounding error of an fp32
evaluation is proportional to.
"""

from __future__ import annotations

import torch
from torch import Tensor

F64 = torch.float64


def d(t):
    """A detached 64-bit CPU copy."""
    return None if t is None else t.detach().to("cpu", F64)


# ----------------------------------------------------------------------------- layer norm
def layer_norm(x: Tensor, w, b, eps: float) -> Tensor:
    xc = x - x.mean(-1, keepdim=True)
    xn = xc / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    return xn * (1 if w is None else w) + (0 if b is None else b)


def layer_norm_mag(x: Tensor, w, b, eps: float) -> Tensor:
    """The mean's error moves a row by rstd * mean|x|, the other steps by their own size."""
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    aw = 1 if w is None else w.abs()
    return aw * (xc.abs() * rstd + rstd * x.abs().mean(-1, keepdim=True)) + (0 if b is None else b.abs())


def layer_norm_grad(dy: Tensor, x: Tensor, w, eps: float) -> tuple:
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xn, g = xc * rstd, dy * (1 if w is None else w)
    dx = rstd * (g - g.mean(-1, keepdim=True) - xn * (g * xn).mean(-1, keepdim=True))
    return dx, (dy * xn).reshape(-1, x.shape[-1]).sum(0), dy.reshape(-1, x.shape[-1]).sum(0)


def layer_norm_grad_mag(dy: Tensor, x: Tensor, w, eps: float) -> tuple:
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    # |xn| with the reach of the mean's error
    xn, g = xc.abs() * rstd + rstd * x.abs().mean(-1, keepdim=True), (dy * (1 if w is None else w)).abs()
    dx = rstd * (g + g.mean(-1, keepdim=True) + xn * (g * xn).mean(-1, keepdim=True))
    return dx, (dy.abs() * xn).reshape(-1, x.shape[-1]).sum(0), dy.abs().reshape(-1, x.shape[-1]).sum(0)


# ----------------------------------------------------------------------------- short conv
def short_conv(x: Tensor, w: Tensor, b, dilation: int, silu: bool, hist=None, lengths=None) -> tuple:
    """``(y, next history)``; x ``[B, T, C]``, w ``[C, K]``, one sequence and position after the other."""
    nb, t, c = x.shape
    k = w.shape[1]
    lp = (k - 1) * dilation
    ys, hs = [], []
    for i in range(nb):
        n = t if lengths is None else max(0, min(t, int(lengths[i])))
        head = x.new_zeros(lp, c) if hist is None else hist[i]
        ext = torch.cat((head, x[i, :n]))
        pre = x.new_zeros(n, c) + (0 if b is None else b)
        for j in range(k):
            pre = pre + w[:, j] * ext[j * dilation:j * dilation + n]
        ys.append(torch.cat((pre * torch.sigmoid(pre) if silu else pre, x.new_zeros(t - n, c))))
        hs.append(ext[n:])
    return torch.stack(ys), torch.stack(hs)


# ----------------------------------------------------------------------------- selective scan
def _decay(s: Tensor, A: Tensor, mag: bool) -> Tensor:
    """``exp(s A)``.  fp32 arithmetic returns zero for an exponential below its smallest normal number 2^-126,
    an error of up to 2^-126 whatever the exponential's size: 2^24 times that in the companion, whose users
    multiply it by at least 2^-24."""
    a = torch.exp(s[..., None] * A)
    return a + 2.0 ** -102 if mag else a


def selective_scan(u, dt, A, B, C, D, z, dt_bias, softplus, state=None, lengths=None, mag=False) -> tuple:
    """``(y, final state)``; B, C ``[B, T, G, N]``.  ``mag``: the same sums of absolute values."""
    nb, t, c = u.shape
    n, rep = A.shape[1], c // B.shape[2]
    ab = (lambda v: v.abs()) if mag else (lambda v: v)
    raw = dt + (0 if dt_bias is None else dt_bias)
    s = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    h = u.new_zeros(nb, c, n) if state is None else ab(state)
    own = torch.full((nb,), t) if lengths is None else lengths.clamp(0, t).to("cpu")
    ys = []
    for i in range(t):
        bi, ci = (ab(v[:, i].repeat_interleave(rep, 1)) for v in (B, C))
        step = _decay(s[:, i], A, mag) * h + ab(s[:, i] * u[:, i])[..., None] * bi
        live = (i < own)[:, None]
        h = torch.where(live[..., None], step, h)
        y = (h * ci).sum(-1) + (0 if D is None else ab(D * u[:, i]))
        if z is not None:
            y = y * ab(z[:, i]) * torch.sigmoid(z[:, i])
        ys.append(torch.where(live, y, torch.zeros_like(y)))
    return (torch.stack(ys, 1) if ys else torch.zeros_like(u)), h


def selective_grad(dy, dend, u, dt, A, B, C, D, z, dt_bias, softplus, state=None, lengths=None, mag=False) -> dict:
    """The gradients by the formulas, one token after the other backwards."""
    nb, t, c = u.shape
    gr, n = B.shape[2], A.shape[1]
    rep = c // gr
    ab = (lambda v: v.abs()) if mag else (lambda v: v)
    raw = dt + (0 if dt_bias is None else dt_bias)
    s = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    own = torch.full((nb,), t) if lengths is None else lengths.clamp(0, t).to("cpu")
    zero = u.new_zeros(())
    hs = [u.new_zeros(nb, c, n) if state is None else ab(state)]
    for i in range(t):
        bi = ab(B[:, i].repeat_interleave(rep, 1))
        step = _decay(s[:, i], A, mag) * hs[-1] + ab(s[:, i] * u[:, i])[..., None] * bi
        hs.append(torch.where((i < own)[:, None, None], step, hs[-1]))
    g = {k: torch.zeros_like(v) for k, v in dict(u=u, dt=dt, A=A, B=B, C=C).items()}
    g["D"], g["dt_bias"] = u.new_zeros(c), u.new_zeros(c)
    g["z"] = torch.zeros_like(u)
    q = u.new_zeros(nb, c, n) if dend is None else ab(dend)
    for i in range(t - 1, -1, -1):
        live = (i < own)[:, None]
        bi, ci = (ab(v[:, i].repeat_interleave(rep, 1)) for v in (B, C))
        a = _decay(s[:, i], A, mag)
        h, hp = hs[i + 1], hs[i]
        ui, si = ab(u[:, i]), ab(s[:, i])
        dyi = torch.where(live, ab(dy[:, i]), zero)
        e = dyi
        if z is not None:
            sg = torch.sigmoid(z[:, i])
            yv = (h * ci).sum(-1) + (0 if D is None else ab(D) * ui)
            slope = sg * (1 + ab(z[:, i]) * (1 - sg))
            g["z"][:, i] = torch.where(live, dyi * yv * slope, zero)
            e = torch.where(live, dyi * ab(z[:, i]) * sg, zero)
        q_in = q + e[..., None] * ci
        gb = (q_in * bi).sum(-1)
        through = q_in * a * hp
        ds = gb * ui + (through * ab(A)).sum(-1)
        if softplus:
            ds = ds * torch.sigmoid(raw[:, i])
        g["u"][:, i] = torch.where(live, gb * si + e * (0 if D is None else ab(D)), zero)
        g["dt"][:, i] = torch.where(live, ds, zero)
        g["dt_bias"] += torch.where(live, ds, zero).sum(0)
        g["A"] += torch.where(live[..., None], through * si[..., None], zero).sum(0)
        g["D"] += torch.where(live, e * ui, zero).sum(0)
        db, dc = q_in * (si * ui)[..., None], h * e[..., None]
        for key, v in (("B", db), ("C", dc)):
            g[key][:, i] = torch.where(live[..., None], v, zero).view(nb, gr, rep, n).sum(2)
        q = torch.where(live[..., None], q_in * a, q)
    g["state"] = q
    return g
