"""The linear attention and group norm entry points refuse what they do not take before any GPU work, and the
modules around them build and load on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lngram_hip import _lib
from lngram_hip.ops import dtype_code

BF, FP = dtype_code(torch.bfloat16), dtype_code(torch.float32)
P = ctypes.c_void_p(4096)


def _args(**change):
    a = _lib.LinearAttention(B=2, T=100, H=4, Hq=4, Hk=2, Hv=2, K=32, V=32, dtype=BF, token_decay=1, scale=1.0)
    for f in ("q", "k", "v", "decay", "state", "y", "state_out", "checkpoints"):
        setattr(a, f, 4096)
    for n, heads in (("q", 4), ("k", 2), ("v", 2)):
        for d, size in (("batch", 100 * heads * 32), ("token", heads * 32), ("head", 32)):
            setattr(a, f"{n}_{d}", size)
    a.decay_batch, a.decay_token = 400, 4
    for k, v in change.items():
        setattr(a, k, v)
    return a


def test_linear_attention_refusals():
    lib = _lib.load()
    assert lib.lng_linear_attention_size() == ctypes.sizeof(_lib.LinearAttention)
    assert lib.lng_linear_attention_grad_size() == ctypes.sizeof(_lib.LinearAttentionGrad)

    def scan(ws=P, n=1 << 40, **kw):
        return lib.lng_linear_attention_scan(ctypes.byref(_args(**kw)), ws, n, None)

    for change, rc in ((dict(dtype=3), -2), (dict(K=0), -1), (dict(K=129), -1), (dict(V=129), -1), (dict(V=0), -1),
                       (dict(H=0), -1), (dict(Hk=3), -1), (dict(Hv=0), -1), (dict(Hq=8), -1), (dict(H=1 << 15), -1),
                       (dict(B=-1), -1), (dict(T=-1), -1), (dict(T=1 << 31), -1), (dict(q=None), -1), (dict(decay=None), -1),
                       (dict(y=None), -1), (dict(B=1 << 20, T=1 << 20), -1)):
        assert scan(**change) == rc, change
        assert b"linear_attention" in lib.lng_last_error()
    assert lib.lng_linear_attention_scan(None, P, 1 << 40, None) == -1
    assert scan(B=0) == 0 and scan(T=0) == 0
    need = lib.lng_linear_attention_workspace_bytes(ctypes.byref(_args(T=5000)), 0)
    assert need > 0 and lib.lng_linear_attention_workspace_bytes(ctypes.byref(_args(K=200)), 0) == 0
    assert lib.lng_linear_attention_workspace_bytes(ctypes.byref(_args(T=5000)), 1) > need
    for ws, n in ((None, need), (P, need - 1), (ctypes.c_void_p(4100), need)):
        assert scan(ws, n, T=5000) == -1
        assert b"workspace" in lib.lng_last_error()
    # rows that are no 16-byte pieces go through the workspace
    assert lib.lng_linear_attention_workspace_bytes(ctypes.byref(_args(T=64, q_token=129)), 0) > 0

    def grad(ws=P, n=1 << 40, g=None, **kw):
        g = g or dict(dy=4096, dy_batch=100 * 128, dy_token=128, dy_head=32, dq=4096, dk=4096, dv=4096, ddecay=4096)
        return lib.lng_linear_attention_scan_grad(ctypes.byref(_args(**kw)), ctypes.byref(_lib.LinearAttentionGrad(**g)), ws, n,
                                                  None)

    assert grad(checkpoints=None) == -1 and grad(B=0) == -1 and grad(g=dict(dy=4096)) == -1
    ok = dict(dy=4096, dy_batch=100 * 128, dy_token=128, dy_head=32, dq=4096, dk=4096, dv=4096, ddecay=4096)
    for change in (dict(dy=4104), dict(dy_token=129), dict(dy_head=33), dict(dy_token=1 << 24)):
        assert grad(g={**ok, **change}) == -1 and b"16-byte" in lib.lng_last_error()
    assert grad(ws=None) == -1 and b"workspace" in lib.lng_last_error()
    assert lib.lng_linear_attention_step(ctypes.byref(_args()), None) == -1 and b"T = 1" in lib.lng_last_error()
    assert lib.lng_linear_attention_step(ctypes.byref(_args(T=1, state=None)), None) == -1
    # launches past 2^32 threads
    assert scan(B=1 << 20, T=1 << 10, H=32, Hq=32) == -1 and b"bad shape" in lib.lng_last_error()
    for kw in (dict(B=1 << 22, T=64, H=8), dict(B=1 << 18, T=1 << 10, H=32, Hq=32),
               dict(B=1 << 12, T=1 << 18, H=1, Hq=1, Hk=1, Hv=1, K=127, V=128)):      # rows through the workspace
        assert scan(**kw) == -1 and b"split the batch" in lib.lng_last_error(), kw
    assert lib.lng_linear_attention_step(ctypes.byref(_args(B=1 << 24, T=1, H=16)), None) == -1
    assert b"split the batch" in lib.lng_last_error()


def test_group_norm_refusals():
    lib = _lib.load()
    names = "x dtype N L C G xs xl w b wt eps silu ws n y mean rstd st".split()
    ok = [P, BF, 4, 100, 64, 8, 6400, 64, P, P, BF, 1e-5, 1, P, 1 << 40, P, P, P, None]

    def call(**kw):
        return lib.lng_group_norm(*[kw.get(n, v) for n, v in zip(names, ok)])

    for kw, rc in ((dict(dtype=3), -2), (dict(wt=2), -2), (dict(N=-1), -1), (dict(L=-1), -1), (dict(C=0), -1), (dict(G=0), -1),
                   (dict(G=7), -1), (dict(x=None), -1), (dict(y=None), -1), (dict(rstd=None), -1), (dict(xs=-64), -1),
                   (dict(N=1 << 30, L=1 << 30), -1)):
        assert call(**kw) == rc, kw
        assert b"group_norm" in lib.lng_last_error()
    assert call(N=0, x=None, y=None) == 0 and call(L=0, x=None, y=None) == 0
    need = lib.lng_group_norm_workspace_bytes(4, 5000, 64, 8, 0)
    assert need > 0 and lib.lng_group_norm_workspace_bytes(0, 1, 64, 8, 0) == 0
    assert lib.lng_group_norm_workspace_bytes(4, 1, 64, 7, 0) == 0
    for ws, n in ((None, need), (P, need - 1), (ctypes.c_void_p(4100), need)):
        assert call(L=5000, ws=ws, n=n) == -1 and b"workspace" in lib.lng_last_error()
    assert call(N=1 << 26, L=1 << 12) == -1 and b"split the batch" in lib.lng_last_error()
    gnames = "dy ds dl x xs xl dtype N L C G w b wt silu mean rstd ws n dx dw db st".split()
    gok = [P, 6400, 64, P, 6400, 64, BF, 4, 100, 64, 8, P, P, BF, 1, P, P, P, 1 << 40, P, P, P, None]

    def grad(**kw):
        return lib.lng_group_norm_grad(*[kw.get(n, v) for n, v in zip(gnames, gok)])

    for kw, rc in ((dict(dy=None), -1), (dict(mean=None), -1), (dict(dl=-1), -1), (dict(ws=None), -1), (dict(n=16), -1),
                   (dict(dtype=5), -2)):
        assert grad(**kw) == rc, kw
    assert grad(N=0, dw=None, db=None) == 0


def test_modules_on_the_cpu():
    from ffnmem.memory.linear_attention import LinearAttentionSSM, linear_attention
    from ffnmem.memory.norm import GroupNorm, group_norm

    n = GroupNorm(4, 16, activation="silu")
    n.load_state_dict(torch.nn.GroupNorm(4, 16).state_dict())
    with pytest.raises(RuntimeError, match="no CPU path"):
        group_norm(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear_attention(*(torch.zeros(1, 2, 1, 4) for _ in range(3)), torch.zeros(1))
    for bad in (lambda: GroupNorm(3, 16), lambda: GroupNorm(4, 16, activation="gelu"), lambda: LinearAttentionSSM(32, 30, 4),
                lambda: LinearAttentionSSM(32, 32, 4, key_dim=129), lambda: LinearAttentionSSM(32, 32, 4, kv_heads=3),
                lambda: LinearAttentionSSM(32, 256, 1), lambda: LinearAttentionSSM(32, decay_max=1.0)):
        with pytest.raises(ValueError):
            bad()
    s = LinearAttentionSSM(32, 64, heads=4, key_dim=8, kv_heads=2)
    assert s.state_dim == 64 and s.empty_state(3).shape == (3, 4, 8, 16) and not hasattr(s, "decay")
    decays = torch.sigmoid(s.decay_bias)
    assert abs(decays[0].item() - 0.5) < 1e-6 and abs(decays[-1].item() - 0.999) < 1e-6
