"""Operators of a block that mixes tokens with a matrix state per head, as measurable cases.

``attn``   linear attention with a decay for each head: prompts (ragged ones that continue from a state too, a few
           drafted tokens) and training
``step``   the same for one new token of every sequence
``gnorm``  group norm with an activation, channels last: one token a sample (each head's output on its own) or whole
           sequences a sample, forward and with its backward pass

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
_CHUNK = 64                                     # tokens of a chunk of the plain form


# ----------------------------------------------------------------------------- the cases
def listed() -> list:
    return [
        # a whole batch of long prompts through the memory layer's head shape, a decay that each token chooses
        {"name": "attn_8x4096x16x64", "kind": "attn", "batch": 8, "seq": 4096, "heads": 16, "q_heads": 16,
         "kv_heads": 16, "key": 64, "value": 64, "dtype": "bf16", "token_decay": True, "start": False, "ragged": False,
         "train": False},
        # one very long prompt: keys and values shared by groups of heads, one decay a head, wide heads
        {"name": "attn_1x16384x16x128", "kind": "attn", "batch": 1, "seq": 16384, "heads": 16, "q_heads": 16,
         "kv_heads": 4, "key": 128, "value": 128, "dtype": "bf16", "token_decay": False, "start": False,
         "ragged": False, "train": False},
        # ragged prompts of an fp32 layer that continue cached ones; odd sizes
        {"name": "attn_ragged_3x777x6", "kind": "attn", "batch": 3, "seq": 777, "heads": 6, "q_heads": 6,
         "kv_heads": 2, "key": 40, "value": 72, "dtype": "fp32", "token_decay": True, "start": True, "ragged": True,
         "train": False},
        # a pending token and four drafted ones of each of 8 sequences, from their states
        {"name": "attn_draft_8x5x16x64", "kind": "attn", "batch": 8, "seq": 5, "heads": 16, "q_heads": 16,
         "kv_heads": 4, "key": 64, "value": 64, "dtype": "bf16", "token_decay": True, "start": True, "ragged": False,
         "train": False},
        # one training step of the scan over whole sequences
        {"name": "attn_train_8x2048x16x64", "kind": "attn", "batch": 8, "seq": 2048, "heads": 16, "q_heads": 16,
         "kv_heads": 16, "key": 64, "value": 64, "dtype": "bf16", "token_decay": True, "start": False, "ragged": False,
         "train": True},
        # a ragged batch of an fp32 layer in training: learned decays a head, shared keys and values
        {"name": "attn_train_ragged_4x500x8", "kind": "attn", "batch": 4, "seq": 500, "heads": 8, "q_heads": 8,
         "kv_heads": 2, "key": 32, "value": 64, "dtype": "fp32", "token_decay": False, "start": True, "ragged": True,
         "train": True},
        # serving: one new token of each of 8 sequences
        {"name": "step_8x16x64", "kind": "step", "batch": 8, "heads": 16, "q_heads": 16, "kv_heads": 4, "key": 64,
         "value": 64, "dtype": "bf16", "token_decay": True},
        # the same for a full batch of sequences: the states come from memory
        {"name": "step_512x16x64", "kind": "step", "batch": 512, "heads": 16, "q_heads": 16, "kv_heads": 16,
         "key": 64, "value": 64, "dtype": "bf16", "token_decay": True},
        # every head's output of a whole batch of prompts normed on its own
        {"name": "gnorm_32768x1024", "kind": "gnorm", "samples": 32768, "len": 1, "groups": 16, "chan": 1024,
         "dtype": "bf16", "act": True, "train": False},
        # whole sequences a sample, few channels a group
        {"name": "gnorm_8x4096x320", "kind": "gnorm", "samples": 8, "len": 4096, "groups": 32, "chan": 320,
         "dtype": "bf16", "act": True, "train": False},
        # one training step's norm of head outputs, weights in fp32 beside bf16 activations
        {"name": "gnorm_train_16384x1024", "kind": "gnorm", "samples": 16384, "len": 1, "groups": 16, "chan": 1024,
         "dtype": "bf16", "weights": "fp32", "act": True, "train": True},
        # the training of a sequence norm without an activation, fp32
        {"name": "gnorm_train_4x1500x256", "kind": "gnorm", "samples": 4, "len": 1500, "groups": 8, "chan": 256,
         "dtype": "fp32", "act": False, "train": True},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], spread over its logarithm."""
    hi = max(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("attn", "attn", "attn", "step", "gnorm", "gnorm"))
    case = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "fp32", "fp16"))}
    if kind == "gnorm":
        train = rng.random() < 0.5
        groups = rng.choice((1, 2, 4, 8, 16, 32))
        chan = groups * _log(rng, 2, 4096 // groups)
        most = (16384 if train else 32768) * 1024 // chan
        length = rng.choice((1, _log(rng, 2, min(most, 65536))))
        samples = _log(rng, 1, min(most // length, 100000))
        case.update(samples=samples, len=length, groups=groups, chan=chan, act=rng.random() < 0.7, train=train)
        if case["dtype"] != "fp32" and rng.random() < 0.5:
            case["weights"] = "fp32"
        return case
    kv = rng.choice((1, 2, 3, 4))
    heads = kv * rng.choice((1, 1, 2, 4))
    case.update(heads=heads, q_heads=rng.choice((heads, heads, kv)), kv_heads=kv,
                key=rng.choice((32, 64, 64, 128, _log(rng, 4, 128))),
                value=rng.choice((32, 64, 64, 128, _log(rng, 4, 128))), token_decay=rng.random() < 0.6)
    size = heads * max(case["key"], case["value"])
    if kind == "step":
        case["batch"] = _log(rng, 1, min(2048, 512 * 16 * 64 * 64 // (heads * case["key"] * case["value"])))
        return case
    train = rng.random() < 0.4
    batch = _log(rng, 1, 8)
    most = (2048 * 8 if train else 4096 * 8) * 16 * 64 // (size * batch)
    case.update(batch=batch, seq=_log(rng, 1, min(4096 if train else 16384, most)), start=rng.random() < 0.5,
                ragged=rng.random() < 0.5, train=train)
    return case


# ----------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6971 + 29)


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32) -> torch.Tensor:
    return torch.empty(*shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=g).to(dtype)


def _lengths(g, batch: int, seq: int) -> torch.Tensor:
    """Lengths of a padded batch of prompts, the longest one full."""
    n = torch.randint(0, seq + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[int(torch.randint(0, batch, (1,), generator=g, device="cuda"))] = seq
    return n


def _head_decays(heads: int) -> torch.Tensor:
    """Log decays a head, their time constants spread geometrically between decays of 0.5 and 0.999."""
    gone = torch.exp(torch.linspace(math.log(0.5), math.log(1e-3), heads, device="cuda"))
    return torch.log1p(-gone)


def _decays(g, case: dict, *lead: int) -> torch.Tensor:
    base = _head_decays(case["heads"])
    if not case["token_decay"]:
        return base
    # a token's own rate: the head's, between a quarter and four times it
    return base * torch.exp(_randn(g, *lead, case["heads"], std=0.7))


def _projected(g, case: dict, *lead: int) -> tuple:
    """q, k and v as parts of the rows of one projection."""
    hq, hk, dk, dv = case["q_heads"], case["kv_heads"], case["key"], case["value"]
    row = _randn(g, *lead, hq * dk + hk * (dk + dv), dtype=_DT[case["dtype"]])
    q, k, v = row.split((hq * dk, hk * dk, hk * dv), dim=-1)
    return q.unflatten(-1, (hq, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hk, dv))


_LEAVES = ("q", "k", "v", "decay", "start")


def prepare(case: dict, seed: int) -> dict:
    kind, dt, g = case["kind"], _DT[case["dtype"]], _gen(seed)
    s = {"case": case}
    if kind == "attn":
        b, t, h, dk, dv = (case[x] for x in ("batch", "seq", "heads", "key", "value"))
        s["q"], s["k"], s["v"] = _projected(g, case, b, t)
        s["decay"] = _decays(g, case, b, t)
        s["start"] = _randn(g, b, h, dk, dv) if case["start"] else None
        s["lengths"] = _lengths(g, b, t) if case["ragged"] else None
        if case["train"]:
            s["dy"], s["dstate"] = _randn(g, b, t, h, dv, dtype=dt), _randn(g, b, h, dk, dv, std=0.1)
            for key in _LEAVES:
                if s[key] is not None:
                    s[key] = s[key].detach().requires_grad_(True)
    elif kind == "step":
        b, h, dk, dv = (case[x] for x in ("batch", "heads", "key", "value"))
        s["q"], s["k"], s["v"] = _projected(g, case, b)
        s["decay"] = _decays(g, case, b)
        # the states of the tokens so far, and those of the next ones: a step that a rejected draft takes back
        # leaves the former as they were
        s["state"] = _randn(g, b, h, dk, dv)
        s["next"] = torch.empty_like(s["state"])
    elif kind == "gnorm":
        n, l, c = case["samples"], case["len"], case["chan"]
        wt = _DT[case.get("weights", case["dtype"])]
        # a group has a mean and a scale of its own, as heads of different horizons do
        scale = torch.exp(_randn(g, case["groups"], 1, std=1.0)).expand(-1, c // case["groups"]).reshape(c)
        x = (_randn(g, n, l, c) * scale + _randn(g, n, 1, c, std=0.5)).to(dt)
        s["x"] = x if l > 1 else x[:, 0]
        s["w"], s["b"] = _randn(g, c, mean=1.0, std=0.2, dtype=wt), _randn(g, c, std=0.2, dtype=wt)
        if case["train"]:
            s["dy"] = _randn(g, *s["x"].shape, dtype=dt)
            for k in ("x", "w", "b"):
                s[k] = s[k].detach().requires_grad_(True)
    else:
        raise ValueError(kind)
    return s


# ----------------------------------------------------------------------------- one pass
def run(s: dict):
    return (_own if own else _plain)(s, s["case"])


def _own(s: dict, case: dict):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    kind = case["kind"]
    if kind == "attn":
        from ffnmem.memory.linear_attention import linear_attention

        y, state = linear_attention(s["q"], s["k"], s["v"], s["decay"], state=s["start"], lengths=s["lengths"],
                                    return_state=True)
        if not case["train"]:
            return {"y": y, "state": state}
        keys = [k for k in _LEAVES if s[k] is not None]
        grads = torch.autograd.grad([y, state], [s[k] for k in keys], [s["dy"], s["dstate"]])
        return {"y": y.detach(), "state": state.detach(), **{"d" + k: v for k, v in zip(keys, grads)}}
    if kind == "step":
        from ffnmem.memory.linear_attention import linear_attention_step

        y = linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["decay"], out_state=s["next"])
        return {"y": y, "state": s["next"]}
    from ffnmem.memory.norm import group_norm

    y = group_norm(s["x"], case["groups"], s["w"], s["b"], _EPS, activation="silu" if case["act"] else None)
    if not case["train"]:
        return y
    dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
    return {"y": y.detach(), "x": dx, "w": dw, "b": db}


# ----------------------------------------------------------------------------- the plain forms, 32 bits
@torch.no_grad()
def _plain(s: dict, case: dict):
    return {"attn": _plain_attn, "step": _plain_step, "gnorm": _plain_gnorm}[case["kind"]](s, case)


def _plain_step(s: dict, case: dict):
    h = case["heads"]
    q, k, v = (s[x].float().repeat_interleave(h // s[x].shape[1], 1) for x in ("q", "k", "v"))
    state = torch.exp(s["decay"])[..., None, None] * s["state"] + k[..., None] * v[:, :, None]
    y = (q[..., None] * state).sum(2) * case["key"] ** -0.5
    s["next"].copy_(state)
    return {"y": y.to(s["q"].dtype), "state": s["next"]}


def _chunks(x: torch.Tensor, heads: int, n: int) -> torch.Tensor:
    """[B, T, h, D] -> [B, H, chunks, _CHUNK, D] in fp32: shared heads repeated, zeros behind the last token."""
    b, t, hx, d = x.shape
    x = x.float().repeat_interleave(heads // hx, 2).transpose(1, 2)
    x = torch.nn.functional.pad(x, (0, 0, 0, n * _CHUNK - t))
    return x.reshape(b, heads, n, _CHUNK, d)


def _unchunk(x: torch.Tensor, t: int) -> torch.Tensor:
    """[B, H, chunks, _CHUNK, D] -> [B, T, H, D]."""
    return x.flatten(2, 3)[:, :, :t].transpose(1, 2)


def _grouped(x: torch.Tensor, heads: int) -> torch.Tensor:
    """The sum over each group of heads that shares one: [B, T, H, D] -> [B, T, heads, D]."""
    return x.unflatten(2, (heads, x.shape[2] // heads)).sum(3)


def _plain_attn(s: dict, case: dict):
    b, t, h, dk, dv = (case[x] for x in ("batch", "seq", "heads", "key", "value"))
    dt, dev, scale = s["q"].dtype, s["q"].device, dk ** -0.5
    n = -(-t // _CHUNK)
    q, k, v = (_chunks(s[x], h, n) for x in ("q", "k", "v"))
    gl = s["decay"].double().expand(b, t, h)[..., None]
    gl = torch.nn.functional.pad(gl.transpose(1, 2), (0, 0, 0, n * _CHUNK - t)).reshape(b, h, n, _CHUNK)
    real = None
    if s["lengths"] is not None:              # behind a sequence's end nothing is added and nothing decays
        real = (torch.arange(n * _CHUNK, device=dev)[None] < s["lengths"][:, None]).view(b, 1, n, _CHUNK)
        q, k, v = (torch.where(real[..., None], x, 0.0) for x in (q, k, v))
        gl = torch.where(real, gl, 0.0)
    # log decays since the chunk's start, and since the sequence's: sums in 64 bits
    inner = gl.cumsum(-1)
    total = inner[..., -1].cumsum(-1)                                        # up to each chunk's end
    start_at = torch.nn.functional.pad(total, (1, 0))[..., :-1]
    low = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=dev).tril()
    dec = torch.exp((inner[..., :, None] - inner[..., None, :]).masked_fill(~low, -math.inf)).float()
    from_start, to_end = torch.exp(inner).float(), torch.exp(inner[..., -1:] - inner).float()
    # what each chunk adds to the state, and the states before the chunks: sums over the chunks before
    before = torch.ones(n, n, dtype=torch.bool, device=dev).tril(-1)
    carry = torch.exp((start_at[..., :, None] - total[..., None, :]).masked_fill(~before, -math.inf)).float()
    add = torch.matmul((k * to_end[..., None]).transpose(-1, -2), v)         # [B, H, n, K, V]
    s_in = torch.matmul(carry, add.flatten(3)).view(b, h, n, dk, dv)
    if s["start"] is not None:
        s_in += torch.exp(start_at).float()[..., None, None] * s["start"][:, :, None]
    qk = torch.matmul(q, k.transpose(-1, -2)) * scale
    y = torch.matmul(qk * dec, v) + torch.matmul(q, s_in) * (from_start * scale)[..., None]
    whole = torch.exp(inner[..., -1]).float()[..., None, None]               # a chunk's decay
    end = whole[:, :, -1] * s_in[:, :, -1] + add[:, :, -1]
    res = {"y": _unchunk(y, t).to(dt), "state": end}
    if not case["train"]:
        return res
    do = _chunks(s["dy"], h, n)
    if real is not None:
        do = torch.where(real[..., None], do, 0.0)
    # the states' gradients behind the chunks: the same sums from the end
    radd = torch.matmul((q * (from_start * scale)[..., None]).transpose(-1, -2), do)
    r_out = torch.matmul(carry.transpose(-1, -2), radd.flatten(3)).view(b, h, n, dk, dv)
    r_out += torch.exp(total[..., -1:] - total).float()[..., None, None] * s["dstate"][:, :, None]
    dov = torch.matmul(do, v.transpose(-1, -2))
    a = dov * dec * scale
    dq_state = torch.matmul(do, s_in.transpose(-1, -2)) * (from_start * scale)[..., None]
    dk_state = torch.matmul(v, r_out.transpose(-1, -2)) * to_end[..., None]
    dq = torch.matmul(a, k) + dq_state
    dk_ = torch.matmul(a.transpose(-1, -2), q) + dk_state
    dv_ = torch.matmul((qk * dec).transpose(-1, -2), do) + torch.matmul(k, r_out) * to_end[..., None]
    # a decay's gradient: every pair and every state that it stands between; the sums within a chunk in 64 bits
    w = (qk * dec * dov).double().tril(-1)
    rows = w.sum(-1) + (q * dq_state).sum(-1)
    cols = w.sum(-2)
    kept = (k * dk_state).sum(-1).double()
    through = (s_in * r_out).sum((-2, -1)).double() * torch.exp(inner[..., -1])
    dg = (rows - cols).flip(-1).cumsum(-1).flip(-1) + (kept.cumsum(-1) - kept) + through[..., None]
    if real is not None:
        dg = torch.where(real, dg, 0.0)
    dg = _unchunk(dg[..., None], t)[..., 0]
    dg = dg if case["token_decay"] else dg.sum((0, 1))
    res.update(dq=_grouped(_unchunk(dq, t), case["q_heads"]).to(dt), dk=_grouped(_unchunk(dk_, t), case["kv_heads"]).to(dt),
               dv=_grouped(_unchunk(dv_, t), case["kv_heads"]).to(dt), ddecay=dg.float())
    if s["start"] is not None:
        res["dstart"] = whole[:, :, 0] * r_out[:, :, 0] + radd[:, :, 0]
    return res


def _plain_gnorm(s: dict, case: dict):
    n, l, gr, c = (case[x] for x in ("samples", "len", "groups", "chan"))
    shape, dt = s["x"].shape, s["x"].dtype
    x = s["x"].float().view(n, l, gr, c // gr)
    w, bias = s["w"].float().view(gr, c // gr), s["b"].float().view(gr, c // gr)
    mean = x.mean((1, 3), keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean((1, 3), keepdim=True) + _EPS)
    xn = xc * rstd
    z = xn * w + bias
    sig = torch.sigmoid(z) if case["act"] else None
    y = (z * sig if case["act"] else z).to(dt).view(shape)
    if not case["train"]:
        return y
    dz = s["dy"].float().view(n, l, gr, c // gr)
    if case["act"]:
        dz = dz * sig * (1 + z * (1 - sig))
    hg = dz * w
    dx = rstd * (hg - hg.mean((1, 3), keepdim=True) - xn * (hg * xn).mean((1, 3), keepdim=True))
    return {"y": y, "x": dx.to(dt).view(shape), "w": (dz * xn).sum((0, 1)).view(c).to(s["w"].dtype),
            "b": dz.sum((0, 1)).view(c).to(s["b"].dtype)}


# ----------------------------------------------------------------------------- the least work
def work(case: dict) -> dict:
    """Each input read once, each output written once; a multiply-add is two operations."""
    es = torch.finfo(_DT[case["dtype"]]).bits // 8
    if case["kind"] == "gnorm":
        n, c = case["samples"] * case["len"] * case["chan"], case["chan"]
        ws = torch.finfo(_DT[case.get("weights", case["dtype"])]).bits // 8
        if case["train"]:     # x and dy in, y and dx out; the weights in, their gradients out
            return {"bytes": 4 * n * es + 4 * c * ws, "flops": n * (8 + 13 + 10 * case["act"])}
        return {"bytes": 2 * n * es + 2 * c * ws, "flops": n * (8 + 4 * case["act"])}
    h, dk, dv = case["heads"], case["key"], case["value"]
    rows = case["batch"] * case.get("seq", 1)
    state = case["batch"] * h * dk * dv * 4
    qkv = rows * (case["q_heads"] * dk + case["kv_heads"] * (dk + dv)) * es
    decay = (rows if case["token_decay"] else 1) * h * 4
    y = rows * h * dv * es
    # a token's state: one product adds to it, one reads it
    flops = rows * h * dk * dv * 4
    if case["kind"] == "step":
        return {"bytes": qkv + decay + y + 2 * state, "flops": flops}
    if case["train"]:         # q, k, v, decays and dy in, their gradients and y out
        return {"bytes": 2 * (qkv + decay + y) + state * (2 + 2 * case["start"]), "flops": flops * 3}
    return {"bytes": qkv + decay + y + state * (1 + case["start"]), "flops": flops}


# ----------------------------------------------------------------------------- the same in 64 bits
@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    return {"attn": _exact_attn, "step": _exact_step, "gnorm": _exact_gnorm}[case["kind"]](case, s, f)


def _exact_step(case, s, f):
    h, b = case["heads"], case["batch"]
    at = {x: torch.arange(h, device="cuda") // (h // f[x].shape[1]) for x in ("q", "k", "v")}
    state = f["state"] * torch.exp(f["decay"].expand(b, h))[..., None, None]
    state += torch.einsum("bhk,bhv->bhkv", f["k"][:, at["k"]], f["v"][:, at["v"]])
    return {"y": torch.einsum("bhk,bhkv->bhv", f["q"][:, at["q"]], state) / math.sqrt(case["key"]), "state": state}


def _exact_attn(case, s, f):
    """Sequence by sequence and head by head as one matrix of weights over all pairs of tokens."""
    b, t, h, dk, dv = (case[x] for x in ("batch", "seq", "heads", "key", "value"))
    scale, train = 1 / math.sqrt(dk), case["train"]
    res = {"y": f["q"].new_zeros(b, t, h, dv), "state": f["q"].new_zeros(b, h, dk, dv)}
    if train:
        for key in _LEAVES:
            if key in f:
                res["d" + key] = torch.zeros_like(f[key])
    lengths = [t] * b if s["lengths"] is None else s["lengths"].tolist()
    for i, m in enumerate(lengths):
        for j in range(h):
            s0 = f["start"][i, j] if "start" in f else f["q"].new_zeros(dk, dv)
            if m == 0:
                res["state"][i, j] = s0
                if train and "start" in f:
                    res["dstart"][i, j] = f["dstate"][i, j]
                continue
            jq, jk = j // (h // case["q_heads"]), j // (h // case["kv_heads"])
            q, k, v = f["q"][i, :m, jq], f["k"][i, :m, jk], f["v"][i, :m, jk]
            at = (f["decay"][i, :m, j] if case["token_decay"] else f["decay"][j].expand(m)).cumsum(0)
            gap = at[:, None] - at[None, :]
            gap.masked_fill_(torch.ones(m, m, dtype=torch.bool, device="cuda").triu(1), -math.inf)
            gap.exp_()
            since, left = torch.exp(at)[:, None], torch.exp(at[-1] - at)[:, None]
            p = torch.mm(q, k.t()).mul_(gap)
            res["y"][i, :m, j] = scale * (torch.mm(p, v) + since * torch.mm(q, s0))
            res["state"][i, j] = torch.mm((k * left).t(), v) + torch.exp(at[-1]) * s0
            if not train:
                continue
            do, de = f["dy"][i, :m, j] * scale, f["dstate"][i, j]
            res["dv"][i, :m, jk] += torch.mm(p.t(), do) + left * torch.mm(k, de)
            a = torch.mm(do, v.t()).mul_(gap)
            del gap
            q_state, k_state = since * torch.mm(do, s0.t()), left * torch.mm(v, de.t())
            res["dq"][i, :m, jq] += torch.mm(a, k) + q_state
            res["dk"][i, :m, jk] += torch.mm(a.t(), q) + k_state
            # by the sum up to each token: a pair's weight grows with the later and falls with the earlier one
            del a
            pair = torch.mm(do, v.t()).mul_(p)
            dat = pair.sum(1) - pair.sum(0) + (q * q_state).sum(1) - (k * k_state).sum(1)
            dat[-1] += (k * k_state).sum() + torch.exp(at[-1]) * (s0 * de).sum()
            dg = dat.flip(0).cumsum(0).flip(0)
            if case["token_decay"]:
                res["ddecay"][i, :m, j] = dg
            else:
                res["ddecay"][j] += dg.sum()
            if "start" in f:
                res["dstart"][i, j] = torch.mm((q * since).t(), do) + torch.exp(at[-1]) * de
    return res


def _exact_gnorm(case, s, f):
    gr, c = case["groups"], case["chan"]
    d = c // gr
    shape = s["x"].shape
    # a group of a sample as one row
    x = f["x"].view(case["samples"], case["len"], gr, d).transpose(1, 2).flatten(2)
    w, bias = (f[k].view(gr, 1, d).expand(gr, case["len"], d).flatten(1) for k in ("w", "b"))
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + _EPS)
    xn = (x - mean) / sd
    z = torch.addcmul(bias, xn, w)
    e = torch.exp(-z)

    def back(v):
        return v.unflatten(2, (case["len"], d)).transpose(1, 2).reshape(shape)

    y = back(z / (1 + e) if case["act"] else z)
    if not case["train"]:
        return y
    dz = f["dy"].view(case["samples"], case["len"], gr, d).transpose(1, 2).flatten(2)
    if case["act"]:
        dz = dz * (1 + e + z * e) / (1 + e) ** 2
    # the Jacobian of a row is (I - 1 1^T / m - xn xn^T / m) / sd
    hg, m = dz * w, x.shape[-1]
    proj = hg.sum(-1, keepdim=True) + xn * (hg * xn).sum(-1, keepdim=True)
    cols = [(v.sum(0).unflatten(1, (case["len"], d)).sum(1)).reshape(c) for v in (dz * xn, dz)]
    return {"y": y, "x": back((hg - proj / m) / sd), "w": cols[0], "b": cols[1]}
