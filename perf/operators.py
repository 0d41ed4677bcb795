"""Operators of a block that mixes tokens with a selective state space, as measurable cases.

``norm``  layer norm over rows, forward and with its backward pass
``conv``  the short causal depthwise convolution with its activation: prompts (ragged ones with a history too)
          and training
``scan``  the selective state space scan: prompts (ragged ones that continue from a state too) and training
``step``  both for one new token of every sequence: the convolution's history and the scan's state move on

``listed()`` holds the named cases, ``draw(rng)`` gives others of the same ranges, ``prepare`` builds what a
program holds before the call, ``run`` is one pass (``own`` false: elementary torch operations; true: this
library's entry points), ``work`` the bytes and operations that a pass cannot do without, and ``exact`` the
same outputs in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "lngram-decode_amd")
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5


# ----------------------------------------------------------------------------- the cases
def listed() -> list:
    return [
        # the pre-norm of a whole batch of hidden states
        {"name": "norm_16384x1024", "kind": "norm", "rows": 16384, "dim": 1024, "dtype": "bf16", "train": False},
        # the memory norm over the route tokens of three odd prompts: many short rows, past every cache
        {"name": "norm_421911x256", "kind": "norm", "rows": 421911, "dim": 256, "dtype": "bf16", "train": False},
        # one training step's norm with its backward, weights in fp32 beside bf16 activations
        {"name": "norm_train_16384x1024", "kind": "norm", "rows": 16384, "dim": 1024, "dtype": "bf16",
         "weights": "fp32", "train": True},
        # the CPU-scale fp32 layer of experiments and tests: launches and latency count
        {"name": "norm_train_512x128", "kind": "norm", "rows": 512, "dim": 128, "dtype": "fp32", "train": True},
        # the token mixer's convolution over a whole batch of long prompts
        {"name": "conv_8x4096x1024", "kind": "conv", "batch": 8, "seq": 4096, "chan": 1024, "taps": 4, "dilation": 1,
         "dtype": "bf16", "history": False, "ragged": False, "train": False},
        # the memory layer's dilated taps over three ragged prompts that continue cached ones
        {"name": "conv_ragged_3x777x1024", "kind": "conv", "batch": 3, "seq": 777, "chan": 1024, "taps": 4,
         "dilation": 3, "dtype": "bf16", "history": True, "ragged": True, "train": False},
        {"name": "conv_train_8x2048x1024", "kind": "conv", "batch": 8, "seq": 2048, "chan": 1024, "taps": 4,
         "dilation": 1, "dtype": "bf16", "history": False, "ragged": False, "train": True},
        # the token router's state features over a whole batch of long sequences: few channels, long rows
        {"name": "scan_8x4096x256", "kind": "scan", "batch": 8, "seq": 4096, "chan": 256, "state": 16, "groups": 1,
         "dtype": "bf16", "start": False, "ragged": False, "train": False},
        # ragged prompts of an fp32 layer that continue cached ones; odd sizes, states shared by channel groups
        {"name": "scan_ragged_3x777x1000", "kind": "scan", "batch": 3, "seq": 777, "chan": 1000, "state": 12,
         "groups": 2, "dtype": "fp32", "start": True, "ragged": True, "train": False},
        # one training step of the scan
        {"name": "scan_train_8x2048x1024", "kind": "scan", "batch": 8, "seq": 2048, "chan": 1024, "state": 16,
         "groups": 1, "dtype": "bf16", "start": False, "ragged": False, "train": True},
        # serving: one new token of each of 8 sequences
        {"name": "step_8x1024", "kind": "step", "batch": 8, "chan": 1024, "state": 16, "groups": 1, "taps": 4,
         "dilation": 1, "dtype": "bf16"},
        # the same for a full batch of sequences: the states come from memory
        {"name": "step_512x2048", "kind": "step", "batch": 512, "chan": 2048, "state": 16, "groups": 1, "taps": 4,
         "dilation": 1, "dtype": "bf16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], spread over its logarithm."""
    hi = max(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("norm", "norm", "conv", "conv", "scan", "scan", "scan", "step"))
    dtype = rng.choice(("bf16", "bf16", "fp32", "fp16"))
    case = {"kind": kind, "dtype": dtype}
    if kind == "norm":
        train = rng.random() < 0.5
        dim = _log(rng, 8, 8192)
        most = (8192 * 1024 if train else 421911 * 256 // 2) // dim
        case.update(rows=_log(rng, 1, min(most, 500000)), dim=dim, train=train)
        if dtype != "fp32" and rng.random() < 0.5:
            case["weights"] = "fp32"
    elif kind == "conv":
        train = rng.random() < 0.4
        chan = _log(rng, 8, 2048)
        batch = _log(rng, 1, 8)
        seq = _log(rng, 1, min(8192, 8 * 2048 * 1024 // (chan * batch)))
        case.update(batch=batch, seq=seq, chan=chan, taps=rng.randint(2, 4), dilation=rng.choice((1, 1, 2, 3)),
                    history=rng.random() < 0.5, ragged=rng.random() < 0.5, train=train)
    elif kind == "scan":
        train = rng.random() < 0.4
        groups = rng.choice((1, 1, 2, 4))
        state = rng.choice((16, 16, _log(rng, 1, 64)))
        chan = groups * _log(rng, 4, 2048 // groups)
        batch = _log(rng, 1, 8)
        seq = _log(rng, 1, min(4096, 8 * 2048 * 1024 * 8 // (chan * batch * state)))
        case.update(batch=batch, seq=seq, chan=chan, state=state, groups=groups, start=rng.random() < 0.5,
                    ragged=rng.random() < 0.5, train=train)
    else:
        groups = rng.choice((1, 1, 2, 4))
        state = rng.choice((16, 16, _log(rng, 1, 64)))
        chan = groups * _log(rng, 4, 2048 // groups)
        case.update(batch=_log(rng, 1, min(512, 512 * 2048 * 16 // (chan * state))), chan=chan, state=state,
                    groups=groups, taps=rng.randint(2, 4), dilation=rng.choice((1, 1, 2, 3)))
    return case


# ----------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 41)


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32) -> torch.Tensor:
    return torch.empty(*shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=g).to(dtype)


def _rand(g, *shape, lo=0.0, hi=1.0) -> torch.Tensor:
    return lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda")


def _lengths(g, batch: int, seq: int) -> torch.Tensor:
    """Lengths of a padded batch of prompts, the longest one full."""
    n = torch.randint(0, seq + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[int(torch.randint(0, batch, (1,), generator=g, device="cuda"))] = seq
    return n


def _scan_weights(g, chan: int, state: int) -> dict:
    """Decay rates -1 .. -state times a channel's own factor; step sizes of 0.001 to 0.1 after the softplus."""
    a = -torch.arange(1, state + 1, device="cuda", dtype=torch.float32) * _rand(g, chan, 1, lo=0.5, hi=1.5)
    step = torch.exp(_rand(g, chan, lo=math.log(1e-3), hi=math.log(1e-1)))
    return {"A": a.contiguous(), "D": _randn(g, chan, mean=1.0, std=0.1), "dt_bias": torch.log(torch.expm1(step))}


def prepare(case: dict, seed: int) -> dict:
    kind, dt, g = case["kind"], _DT[case["dtype"]], _gen(seed)
    s = {"case": case}
    if kind == "norm":
        # hidden states with a mean of their own per row, as a residual stream has
        n, d = case["rows"], case["dim"]
        wt = _DT[case.get("weights", case["dtype"])]
        s["x"] = (_randn(g, n, d) + _randn(g, n, 1, std=0.5)).to(dt)
        s["w"], s["b"] = _randn(g, d, mean=1.0, std=0.2, dtype=wt), _randn(g, d, std=0.2, dtype=wt)
        if case["train"]:
            s["dy"] = _randn(g, n, d, dtype=dt)
            for k in ("x", "w", "b"):
                s[k].requires_grad_(True)
    elif kind == "conv":
        b, t, c, k, dil = (case[x] for x in ("batch", "seq", "chan", "taps", "dilation"))
        # the mixer's input is one half of a projection's output: rows twice as long as the channels
        s["x"] = _randn(g, b, t, 2 * c, dtype=dt)[..., :c]
        s["w"], s["b"] = _randn(g, c, k, std=0.5, dtype=dt), _randn(g, c, std=0.2, dtype=dt)
        s["hist"] = _randn(g, b, (k - 1) * dil, c, dtype=dt) if case["history"] else None
        s["lengths"] = _lengths(g, b, t) if case["ragged"] else None
        if case["train"]:
            s["dy"] = _randn(g, b, t, c, dtype=dt)
            for key in ("x", "w", "b", "hist"):
                if s[key] is not None:
                    s[key] = s[key].requires_grad_(True)
    elif kind == "scan":
        b, t, c, n, gr = (case[x] for x in ("batch", "seq", "chan", "state", "groups"))
        s.update(_scan_weights(g, c, n))
        s["u"], s["dt"] = _randn(g, b, t, c, dtype=dt), _randn(g, b, t, c, std=0.5, dtype=dt)
        # the gate is the other half of the projection's output, B and C are parts of one row
        s["z"] = _randn(g, b, t, 2 * c, dtype=dt)[..., c:]
        bc = _randn(g, b, t, 2 * gr * n, dtype=dt)
        s["B"], s["C"] = (v.unflatten(-1, (gr, n)) for v in bc.split(gr * n, dim=-1))
        s["start"] = _randn(g, b, c, n, std=0.5) if case["start"] else None
        s["lengths"] = _lengths(g, b, t) if case["ragged"] else None
        if case["train"]:
            s["dy"], s["dstate"] = _randn(g, b, t, c, dtype=dt), _randn(g, b, c, n, std=0.1)
            for key in _SCAN_LEAVES:
                if s[key] is not None:
                    s[key] = s[key].detach().requires_grad_(True)
    elif kind == "step":
        b, c, n, gr, k, dil = (case[x] for x in ("batch", "chan", "state", "groups", "taps", "dilation"))
        s.update(_scan_weights(g, c, n))
        s["w"], s["b"] = _randn(g, c, k, std=0.5, dtype=dt), _randn(g, c, std=0.2, dtype=dt)
        xz = _randn(g, b, 2 * c, dtype=dt)
        s["x"], s["z"] = xz[:, :c], xz[:, c:]
        # a layer's scan reads the convolution through a projection: an input of its own here, so that a
        # rounding of the one is not an input of the other
        s["u"], s["dt"] = _randn(g, b, c, dtype=dt), _randn(g, b, c, std=0.5, dtype=dt)
        bc = _randn(g, b, 2 * gr * n, dtype=dt)
        s["B"], s["C"] = (v.unflatten(-1, (gr, n)) for v in bc.split(gr * n, dim=-1))
        # the caches of the tokens so far, and those of the next ones: a step that a rejected draft takes
        # back leaves the former as they were
        s["hist"] = _randn(g, b, (k - 1) * dil, c, dtype=dt)
        s["state"] = _randn(g, b, c, n, std=0.5)
        s["next_hist"], s["next_state"] = torch.empty_like(s["hist"]), torch.empty_like(s["state"])
    else:
        raise ValueError(kind)
    return s


_SCAN_LEAVES = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "start")


# ----------------------------------------------------------------------------- one pass
def run(s: dict):
    return (_own if own else _plain)(s, s["case"])


def _own(s: dict, case: dict):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    kind = case["kind"]
    if kind == "norm":
        from ffnmem.memory.norm import layer_norm

        y = layer_norm(s["x"], s["w"], s["b"], _EPS)
        if not case["train"]:
            return y
        dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
        return {"y": y.detach(), "x": dx, "w": dw, "b": db}
    if kind == "conv":
        from ffnmem.memory.short_conv import short_conv

        y, hist = short_conv(s["x"], s["w"], s["b"], dilation=case["dilation"], activation="silu", history=s["hist"],
                             lengths=s["lengths"], return_history=True)
        if not case["train"]:
            return {"y": y, "hist": hist}
        keys = [k for k in ("x", "w", "b", "hist") if s[k] is not None]
        return {"y": y.detach(), **dict(zip(keys, torch.autograd.grad(y, [s[k] for k in keys], s["dy"])))}
    if kind == "scan":
        from ffnmem.memory.selective import selective_scan

        y, state = selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                  dt_softplus=True, state=s["start"], lengths=s["lengths"], return_state=True)
        if not case["train"]:
            return {"y": y, "state": state}
        keys = [k for k in _SCAN_LEAVES if s[k] is not None]
        grads = torch.autograd.grad([y, state], [s[k] for k in keys], [s["dy"], s["dstate"]])
        return {"y": y.detach(), "state": state.detach(), **{"d" + k: v for k, v in zip(keys, grads)}}
    from ffnmem.memory.selective import selective_step
    from ffnmem.memory.short_conv import short_conv_step

    conv = short_conv_step(s["x"], s["hist"], s["w"], s["b"], dilation=case["dilation"], activation="silu",
                           out_history=s["next_hist"])
    y = selective_step(s["state"], s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                       dt_softplus=True, out_state=s["next_state"])
    return {"conv": conv, "y": y, "hist": s["next_hist"], "state": s["next_state"]}


# ----------------------------------------------------------------------------- the plain forms, 32 bits
@torch.no_grad()
def _plain(s: dict, case: dict):
    kind = case["kind"]
    if kind == "norm":
        return _plain_norm(s, case)
    if kind == "conv":
        return _plain_conv(s, case)
    if kind == "scan":
        return _plain_scan(s, case)
    # one token: the convolution's window is the history and the new row
    f = {k: v.float() for k, v in s.items() if isinstance(v, torch.Tensor)}
    dil, gr, dt = case["dilation"], case["groups"], s["x"].dtype
    win = torch.cat((f["hist"], f["x"][:, None]), 1)
    pre = (win[:, ::dil] * f["w"].t()).sum(1) + f["b"]
    conv = (pre * torch.sigmoid(pre)).to(dt)
    uf = f["u"]
    step = _softplus(f["dt"] + f["dt_bias"])
    rep = case["chan"] // gr
    bm, cm = (f[k].repeat_interleave(rep, 1) for k in ("B", "C"))
    state = torch.exp(step[..., None] * f["A"]) * f["state"] + (step * uf)[..., None] * bm
    y = (state * cm).sum(-1) + f["D"] * uf
    y = y * f["z"] * torch.sigmoid(f["z"])
    s["next_hist"].copy_(torch.cat((s["hist"], s["x"][:, None]), 1)[:, 1:])
    s["next_state"].copy_(state)
    return {"conv": conv, "y": y.to(dt), "hist": s["next_hist"], "state": s["next_state"]}


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _real(lengths, t: int, device) -> torch.Tensor | None:
    """[B, T, 1] true at a sequence's own positions."""
    if lengths is None:
        return None
    return (torch.arange(t, device=device)[None] < lengths[:, None])[..., None]


def _plain_norm(s: dict, case: dict):
    x, w = s["x"].float(), s["w"].float()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + _EPS)
    xn = xc * rstd
    y = (xn * w + s["b"].float()).to(s["x"].dtype)
    if not case["train"]:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xn * (g * xn).mean(-1, keepdim=True))
    return {"y": y, "x": dx.to(y.dtype), "w": (dy * xn).sum(0).to(s["w"].dtype), "b": dy.sum(0).to(s["b"].dtype)}


def _plain_conv(s: dict, case: dict):
    b, t, c, k, dil = (case[x] for x in ("batch", "seq", "chan", "taps", "dilation"))
    lp, dt = (k - 1) * dil, s["x"].dtype
    real = _real(s["lengths"], t, s["x"].device)
    x = s["x"].float()
    if real is not None:
        x = torch.where(real, x, 0.0)
    head = x.new_zeros(b, lp, c) if s["hist"] is None else s["hist"].float()
    ext = torch.cat((head, x), 1)                                # position p of a sequence at row lp + p
    w = s["w"].float()
    pre = sum(ext[:, j * dil:j * dil + t] * w[:, j] for j in range(k)) + s["b"].float()
    sig = torch.sigmoid(pre)
    y = pre * sig
    if real is not None:
        y = torch.where(real, y, 0.0)
    y = y.to(dt)
    if not case["train"]:
        n = torch.full((b,), t, device=x.device) if s["lengths"] is None else s["lengths"].long()
        at = n[:, None] + torch.arange(lp, device=x.device)
        hist = torch.gather(ext, 1, at[..., None].expand(b, lp, c)).to(dt)
        return {"y": y, "hist": hist}
    dpre = s["dy"].float() * sig * (1 + pre * (1 - sig))
    if real is not None:
        dpre = torch.where(real, dpre, 0.0)
    dext = torch.zeros_like(ext)
    dw = torch.empty_like(w)
    for j in range(k):
        dext[:, j * dil:j * dil + t] += dpre * w[:, j]
        dw[:, j] = (dpre * ext[:, j * dil:j * dil + t]).sum((0, 1))
    dx = dext[:, lp:]
    if real is not None:
        dx = torch.where(real, dx, 0.0)
    out = {"y": y, "x": dx.to(dt), "w": dw.to(s["w"].dtype), "b": dpre.sum((0, 1)).to(s["b"].dtype)}
    if s["hist"] is not None:
        out["hist"] = dext[:, :lp].to(dt)
    return out


def _plain_scan(s: dict, case: dict):
    b, t, c, n, gr = (case[x] for x in ("batch", "seq", "chan", "state", "groups"))
    rep, dt = c // gr, s["u"].dtype
    real = _real(s["lengths"], t, s["u"].device)
    u, z = s["u"].float(), s["z"].float()
    raw = s["dt"].float() + s["dt_bias"]
    step = _softplus(raw)
    if real is not None:                                          # no time passes behind a sequence's end
        step = torch.where(real, step, 0.0)
    # [T, B, ...] so that a time step is one contiguous block
    bm, cm = (s[k].float().transpose(0, 1) for k in ("B", "C"))   # [T, B, G, N]
    shape = (t, b, gr, rep, n)
    step_t, u_t = (v.transpose(0, 1).reshape(t, b, gr, rep, 1) for v in (step, u))
    a = s["A"].view(gr, rep, n)
    decay = torch.exp(step_t * a)
    h = (step_t * u_t) * bm[:, :, :, None]                        # what each step adds, then the states
    start = u.new_zeros(b, gr, rep, n) if s["start"] is None else s["start"].view(b, gr, rep, n)
    prev = start
    for i in range(t):
        h[i].addcmul_(decay[i], prev)
        prev = h[i]
    y_t = (h * cm[:, :, :, None]).sum(-1)
    y = y_t.reshape(t, b, c).transpose(0, 1) + s["D"] * u
    sig = torch.sigmoid(z)
    gate = z * sig
    out = y * gate
    if real is not None:
        out = torch.where(real, out, 0.0)
    res = {"y": out.to(dt), "state": prev.reshape(b, c, n).clone()}
    if not case["train"]:
        return res
    dy = s["dy"].float()
    if real is not None:
        dy = torch.where(real, dy, 0.0)
    dz = dy * y * sig * (1 + z * (1 - sig))
    dyg = dy * gate
    dyg_t = dyg.transpose(0, 1).reshape(t, b, gr, rep, 1)
    dcm = (h * dyg_t).sum(3)
    gh = dyg_t * cm[:, :, :, None]                                # what each output adds, then the states' gradients
    nxt = s["dstate"].view(b, gr, rep, n)
    gh[t - 1] += nxt
    for i in range(t - 2, -1, -1):
        gh[i].addcmul_(decay[i + 1], gh[i + 1])
    dbm = (gh * (step_t * u_t)).sum(3)
    gb = (gh * bm[:, :, :, None]).sum(-1, keepdim=True)
    du = (gb * step_t).reshape(t, b, c).transpose(0, 1) + dyg * s["D"]
    gh *= decay
    dstart = gh[0].reshape(b, c, n).clone()
    gh[1:] *= h[:-1]
    gh[0] *= start
    dstep = (gb * u_t).reshape(t, b, c) + (gh * a).sum(-1).reshape(t, b, c)
    da = (gh * step_t).sum((0, 1)).reshape(c, n)
    ddt = dstep.transpose(0, 1) * torch.sigmoid(raw)
    if real is not None:
        ddt, du, dz = (torch.where(real, v, 0.0) for v in (ddt, du, dz))
        m = real.transpose(0, 1)[..., None]
        dbm, dcm = (torch.where(m, v, 0.0) for v in (dbm, dcm))
    res.update(du=du.to(dt), ddt=ddt.to(dt), dA=da, dB=dbm.transpose(0, 1).to(dt), dC=dcm.transpose(0, 1).to(dt),
               dD=(dyg * u).sum((0, 1)), dz=dz.to(dt), ddt_bias=ddt.sum((0, 1)))
    if s["start"] is not None:
        res["dstart"] = dstart
    return res


# ----------------------------------------------------------------------------- the least work
def work(case: dict) -> dict:
    """Each input read once, each output written once; a multiply-add is two operations, an exponential one."""
    es = torch.finfo(_DT[case["dtype"]]).bits // 8
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["dim"]
        ws = torch.finfo(_DT[case.get("weights", case["dtype"])]).bits // 8
        if case["train"]:     # x and dy in, y and dx out; the weights in, their gradients out
            return {"bytes": 4 * n * es + 4 * case["dim"] * ws, "flops": 8 * n + 13 * n}
        return {"bytes": 2 * n * es + 2 * case["dim"] * ws, "flops": 8 * n}
    if kind == "conv":
        b, t, c, k, dil = (case[x] for x in ("batch", "seq", "chan", "taps", "dilation"))
        n, hist, wts = b * t * c, b * (k - 1) * dil * c, c * (k + 1)
        if case["train"]:
            return {"bytes": (4 * n + 2 * hist * case["history"] + 2 * wts) * es, "flops": n * (2 * k + 4 + 4 * k + 10)}
        return {"bytes": (2 * n + hist * (1 + case["history"]) + wts) * es, "flops": n * (2 * k + 4)}
    gr, st = case["groups"], case["state"]
    if kind == "scan":
        b, t, c = case["batch"], case["seq"], case["chan"]
        n, bc, state, wts = b * t * c, 2 * b * t * gr * st, b * c * st * 4, (c * st + 2 * c) * 4
        if case["train"]:     # u, dt, z, dy in, y and three gradients out; B and C in, their gradients out
            return {"bytes": (8 * n + 2 * bc) * es + state * (2 + 2 * case["start"]) + 2 * wts,
                    "flops": n * (st * (8 + 18) + 40)}
        return {"bytes": (4 * n + bc) * es + state * (1 + case["start"]) + wts, "flops": n * (st * 8 + 15)}
    b, c, k, dil = (case[x] for x in ("batch", "chan", "taps", "dilation"))
    n, hist = b * c, b * (k - 1) * dil * c
    return {"bytes": (6 * n + 2 * b * gr * st + 2 * hist + c * (k + 1)) * es + 2 * n * st * 4 + (c * st + 2 * c) * 4,
            "flops": n * (2 * k + 4 + 8 * st + 15)}


# ----------------------------------------------------------------------------- the same in 64 bits
@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan, "step": _exact_step}[case["kind"]](case, s, f)


def _exact_norm(case, s, f):
    x, d = f["x"], case["dim"]
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + _EPS)
    xn = (x - mean) / sd
    y = torch.addcmul(f["b"], xn, f["w"])
    if not case["train"]:
        return y
    # the Jacobian of a row is (I - 1 1^T / d - xn xn^T / d) / sd
    g = f["dy"] * f["w"]
    proj = g.sum(-1, keepdim=True) + xn * (g * xn).sum(-1, keepdim=True)
    return {"y": y, "x": (g - proj / d) / sd, "w": torch.einsum("nd,nd->d", f["dy"], xn), "b": f["dy"].sum(0)}


def _tokens(s, b: int, t: int) -> list:
    return [t] * b if s["lengths"] is None else s["lengths"].tolist()


def _exact_conv(case, s, f):
    b, t, c, k, dil = (case[x] for x in ("batch", "seq", "chan", "taps", "dilation"))
    lp = (k - 1) * dil
    y = f["x"].new_zeros(b, t, c)
    hist = f["x"].new_zeros(b, lp, c)
    dx, dh = torch.zeros_like(y), torch.zeros_like(hist)
    dw, db = f["x"].new_zeros(c, k), f["x"].new_zeros(c)
    for i, n in enumerate(_tokens(s, b, t)):                      # one sequence after the other, its own length
        rows = torch.cat((f["hist"][i] if "hist" in f else f["x"].new_zeros(lp, c), f["x"][i, :n]))
        hist[i] = rows[n:]
        if n == 0:
            continue
        taps = rows.unfold(0, lp + 1, 1)[..., ::dil]              # [n, C, K]
        pre = (taps * f["w"]).sum(-1) + f["b"]
        e = torch.exp(-pre)
        y[i, :n] = pre / (1 + e)
        if case["train"]:
            dp = f["dy"][i, :n] * (1 + e + pre * e) / (1 + e) ** 2
            dw += (taps * dp[..., None]).sum(0)
            db += dp.sum(0)
            dr = torch.zeros_like(rows)
            for j in range(k):
                dr[j * dil:j * dil + n] += dp * f["w"][:, j]
            dh[i], dx[i, :n] = dr[:lp], dr[lp:]
        # a history's rows of a sequence of no tokens pass through and get no gradient from the outputs
    if not case["train"]:
        return {"y": y, "hist": hist}
    out = {"y": y, "x": dx, "w": dw, "b": db}
    if "hist" in f:
        out["hist"] = dh
    return out


def _doubling(a: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """``h[t] = a[t] h[t-1] + v[t]`` over the first axis by doubling: after a pass of width w every element
    holds its own and the 2w - 1 elements before it."""
    w, n = 1, v.shape[0]
    while w < n:
        nv, na = v.clone(), a.clone()
        nv[w:] += a[w:] * v[:-w]
        na[w:] *= a[:-w]
        v, a, w = nv, na, 2 * w
    return v


def _exact_scan(case, s, f):
    b, t, c, n, gr = (case[x] for x in ("batch", "seq", "chan", "state", "groups"))
    rep = c // gr
    res = {"y": f["u"].new_zeros(b, t, c), "state": f["u"].new_zeros(b, c, n)}
    if case["train"]:
        for k in _SCAN_LEAVES:
            if k in f:
                res["d" + k] = torch.zeros_like(f[k])
    A = f["A"]
    for i, m in enumerate(_tokens(s, b, t)):                      # one sequence after the other, its own length
        h0 = f["start"][i] if "start" in f else A.new_zeros(c, n)
        if m == 0:
            res["state"][i] = h0
            if case["train"] and "start" in f:
                res["dstart"][i] = f["dstate"][i]
            continue
        u, z, raw = f["u"][i, :m], f["z"][i, :m], f["dt"][i, :m] + f["dt_bias"]
        step = torch.logaddexp(raw, torch.zeros_like(raw))
        bm, cm = (f[k][i, :m].repeat_interleave(rep, 1) for k in ("B", "C"))      # [m, C, N]
        dec = torch.exp(step[..., None] * A)
        v = (step * u)[..., None] * bm
        v[0] += dec[0] * h0
        h = _doubling(dec, v)
        y = torch.einsum("tcn,tcn->tc", h, cm) + f["D"] * u
        e = torch.exp(-z)
        res["y"][i, :m], res["state"][i] = y * z / (1 + e), h[-1]
        if not case["train"]:
            continue
        dy = f["dy"][i, :m]
        dys = dy * z / (1 + e)
        res["dz"][i, :m] = dy * y * (1 + e + z * e) / (1 + e) ** 2
        # the states' gradients run backwards: g[t] = C[t] dys[t] + decay[t+1] g[t+1]
        gv = cm * dys[..., None]
        gv[-1] += f["dstate"][i]
        back = torch.cat((torch.zeros_like(dec[:1]), dec.flip(0)[:-1]))
        gs = _doubling(back, gv.flip(0)).flip(0)
        before = torch.cat((h0[None], h[:-1]))
        through = gs * dec * before                                # d(decay) times decay
        gb = torch.einsum("tcn,tcn->tc", gs, bm)
        res["du"][i, :m] = gb * step + dys * f["D"]
        draw_ = (gb * u + torch.einsum("tcn,cn->tc", through, A)) / (1 + torch.exp(-raw))
        res["ddt"][i, :m] = draw_
        res["ddt_bias"] += draw_.sum(0)
        res["dA"] += torch.einsum("tcn,tc->cn", through, step)
        res["dD"] += (dys * u).sum(0)
        res["dB"][i, :m] = (gs * (step * u)[..., None]).view(m, gr, rep, n).sum(2)
        res["dC"][i, :m] = (h * dys[..., None]).view(m, gr, rep, n).sum(2)
        if "start" in f:
            res["dstart"][i] = gs[0] * dec[0]
    return res


def _exact_step(case, s, f):
    dil, rep = case["dilation"], case["chan"] // case["groups"]
    rows = torch.cat((f["hist"], f["x"][:, None]), 1)
    pre = torch.einsum("bkc,ck->bc", rows[:, ::dil], f["w"]) + f["b"]
    conv, uf = pre / (1 + torch.exp(-pre)), f["u"]
    step = torch.logaddexp(f["dt"] + f["dt_bias"], torch.zeros_like(uf))
    bm, cm = (f[k].repeat_interleave(rep, 1) for k in ("B", "C"))
    state = f["state"] * torch.exp(step[..., None] * f["A"]) + bm * (step * uf)[..., None]
    y = (torch.einsum("bcn,bcn->bc", state, cm) + f["D"] * uf) * f["z"] / (1 + torch.exp(-f["z"]))
    return {"conv": conv, "y": y, "hist": rows[:, 1:], "state": state}
