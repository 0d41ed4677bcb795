"""The norm, short conv and selective scan entry points refuse what they do not take before any GPU work,
and the modules around them build and load on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lngram_hip import _lib
from lngram_hip.ops import dtype_code

BF, FP = dtype_code(torch.bfloat16), dtype_code(torch.float32)
P = ctypes.c_void_p(4096)


def test_layer_norm_refusals():
    lib = _lib.load()
    ok = [P, BF, 4, 64, 64, P, P, BF, 1e-5, P, P, P, None]

    def call(**kw):
        names = "x dtype rows d xs w b wt eps y mean rstd st".split()
        return lib.lng_layer_norm(*[kw.get(n, v) for n, v in zip(names, ok)])

    for kw, rc in ((dict(dtype=3), -2), (dict(wt=2), -2), (dict(rows=-1), -1), (dict(d=0), -1), (dict(x=None), -1),
                   (dict(y=None), -1), (dict(rstd=None), -1), (dict(xs=-64), -1)):
        assert call(**kw) == rc, kw
        assert b"layer_norm" in lib.lng_last_error()
    assert call(rows=0, x=None, y=None) == 0
    need = lib.lng_layer_norm_grad_workspace_bytes(1000, 64)
    assert need > 0 and lib.lng_layer_norm_grad_workspace_bytes(0, 64) == 0
    for ws, n in ((None, need), (P, need - 1), (ctypes.c_void_p(4100), need)):
        assert lib.lng_layer_norm_grad(P, 64, P, 64, BF, 1000, 64, P, BF, P, P, ws, n, P, P, P, None) == -1
        assert b"workspace" in lib.lng_last_error()


def test_short_conv_refusals():
    lib = _lib.load()
    names = "x dtype B T C xb xt w bias wt K dil silu hist lengths y hist_out st".split()
    ok = [P, BF, 2, 8, 16, 128, 16, P, P, BF, 4, 1, 1, P, None, P, ctypes.c_void_p(8192), None]

    def call(**kw):
        return lib.lng_short_conv(*[kw.get(n, v) for n, v in zip(names, ok)])

    for kw, rc in ((dict(dtype=3), -2), (dict(wt=2), -2), (dict(K=0), -1), (dict(K=9), -1), (dict(dil=0), -1),
                   (dict(silu=2), -1), (dict(C=0), -1), (dict(B=-1), -1), (dict(T=1 << 40), -1), (dict(x=None), -1),
                   (dict(w=None), -1), (dict(hist_out=P), -1)):
        assert call(**kw) == rc, kw
        assert b"short_conv" in lib.lng_last_error()
    assert call(B=0) == 0 and call(T=0, hist_out=None) == 0
    need = lib.lng_short_conv_grad_workspace_bytes(2, 8, 16, 4, 1)
    assert need > 0
    assert lib.lng_short_conv_grad(P, 128, 16, P, 128, 16, BF, 2, 8, 16, P, P, BF, 4, 1, 1, None, None, None, P, need - 1,
                                   P, P, P, None, None) == -1
    assert lib.lng_short_conv_step(P, BF, 2, 16, 16, P, P, BF, 4, 1, 1, None, P, P, None) == -1


def _args(**change):
    a = _lib.Selective(B=2, T=8, C=16, N=4, G=1, dtype=FP, softplus=1)
    for f in ("u", "dt", "z", "Bm", "Cm", "A", "y", "state", "state_out"):
        setattr(a, f, 4096)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def test_selective_refusals():
    lib = _lib.load()
    assert lib.lng_selective_size() == ctypes.sizeof(_lib.Selective)
    assert lib.lng_selective_grad_size() == ctypes.sizeof(_lib.SelectiveGrad)
    need = lib.lng_selective_workspace_bytes(2, 8, 16, 4, 1, 0)
    assert 0 < need <= lib.lng_selective_workspace_bytes(2, 8, 16, 4, 1, 1)
    assert lib.lng_selective_workspace_bytes(2, 8, 16, 300, 1, 0) == 0
    for change, rc in ((dict(dtype=3), -2), (dict(N=0), -1), (dict(N=257), -1), (dict(G=3), -1), (dict(G=0), -1),
                       (dict(C=-1), -1), (dict(T=-1), -1), (dict(u=None), -1), (dict(A=None), -1), (dict(y=None), -1),
                       (dict(B=1 << 24, T=1 << 20), -1)):
        assert lib.lng_selective_scan(ctypes.byref(_args(**change)), P, 1 << 40, None) == rc, change
        assert b"selective_scan" in lib.lng_last_error()
    for ws, n in ((None, need), (P, need - 1), (ctypes.c_void_p(4100), need)):
        assert lib.lng_selective_scan(ctypes.byref(_args()), ws, n, None) == -1
    assert lib.lng_selective_scan(None, P, need, None) == -1
    assert lib.lng_selective_scan(ctypes.byref(_args(B=0)), None, 0, None) == 0
    g = _lib.SelectiveGrad(dy=4096, du=4096, ddt=4096, dB=4096, dC=4096)
    assert lib.lng_selective_scan_grad(ctypes.byref(_args(checkpoints_in=4096)), ctypes.byref(g), P, 1 << 40, None) == -1  # z without dz
    assert lib.lng_selective_scan_grad(ctypes.byref(_args()), ctypes.byref(g), P, 1 << 40, None) == -1  # no checkpoints
    assert lib.lng_selective_step(ctypes.byref(_args()), None) == -1 and b"T = 1" in lib.lng_last_error()
    assert lib.lng_selective_step(ctypes.byref(_args(T=1, state=None)), None) == -1


def test_modules_on_the_cpu():
    from ffnmem.memory.lngram_v2 import RouteNgramMemoryV2, build_lngram_norm
    from ffnmem.memory.norm import layer_norm
    from ffnmem.memory.selective import SelectiveSSM

    n = build_lngram_norm("LayerNorm", 8, 1e-6)
    n.load_state_dict(torch.nn.LayerNorm(8).state_dict())
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(torch.zeros(2, 8))
    m = RouteNgramMemoryV2(64, num_routes=4, memory_dim=16, readout_num_heads=4, readout_num_kv_heads=2,
                           readout_head_dim=16, normalization="LayerNorm", conv_bias=True)
    assert {"readout_query_norm.bias", "short_conv.norm.bias", "short_conv.conv.bias"} <= set(m.state_dict())
    s = SelectiveSSM(32, 16)
    assert s.state_dim == 16 and s.dt_rank == 2
    steps = torch.nn.functional.softplus(s.dt_bias)
    assert float(steps.min()) > 0.9e-3 and float(steps.max()) < 0.11
    with pytest.raises(ValueError):
        SelectiveSSM(32, 16, conv_kernel=9)
    with pytest.raises(ValueError):
        SelectiveSSM(32, 16, dt_min=0.0)


def test_launches_past_2_to_the_32_threads_are_refused():
    """A launch's blocks times threads are counted in 32 bits: a call that any of its launches would take past them
    is refused before the first one."""
    lib = _lib.load()
    ws = ctypes.c_void_p(4096)
    grads = _lib.SelectiveGrad(dy=4096, du=4096, ddt=4096, dz=4096, dB=4096, dC=4096)

    def scan(**kw):
        return lib.lng_selective_scan(ctypes.byref(_args(**kw)), ws, 1 << 50, None)

    def grad(**kw):
        return lib.lng_selective_scan_grad(ctypes.byref(_args(checkpoints_in=4096, **kw)), ctypes.byref(grads), ws, 1 << 50,
                                           None)

    def step(**kw):
        return lib.lng_selective_step(ctypes.byref(_args(T=1, **kw)), None)

    calls = [lambda: scan(B=1 << 12, T=1 << 12, C=1, N=256),             # a value of B and C a thread
             lambda: scan(B=1 << 12, T=1 << 12, C=16, G=16, N=16),
             lambda: scan(B=1 << 20, T=1, C=1 << 13, N=1),               # a channel a lane
             lambda: grad(B=1 << 12, T=1 << 11, C=1, N=256),             # dB and dC: a thread each
             lambda: grad(B=1 << 20, T=1 << 10, C=64, N=4),
             lambda: step(B=1 << 20, C=1 << 12, N=16),                   # four lanes a channel
             lambda: step(B=1 << 20, C=1 << 12, N=1)]
    for i, call in enumerate(calls):
        assert call() == -1, i
        assert b"split the batch" in lib.lng_last_error(), i

    names = "x dtype B T C xb xt w bias wt K dil silu hist lengths y hist_out st".split()
    ok = [P, BF, 2, 8, 16, 128, 16, P, P, BF, 4, 1, 1, P, None, P, ctypes.c_void_p(8192), None]
    for kw in (dict(B=1, T=1 << 31, C=31, xb=0, xt=31, K=8),             # a channel a thread, four positions
               dict(B=1 << 21, T=17, C=1501, xb=17 * 1501, xt=1501, hist_out=None),  # sixteen, in two tiles
               dict(B=1 << 11, T=0, C=1024, K=8, dil=4096, hist=None),   # the next history alone: a thread a channel
               dict(B=1 << 12, T=1, C=1023, K=8, dil=2048, xb=1023, xt=1023)):
        assert lib.lng_short_conv(*[kw.get(n, v) for n, v in zip(names, ok)]) == -1, kw
        assert b"split the batch" in lib.lng_last_error(), kw
    assert lib.lng_short_conv_step(P, BF, 1 << 20, (1 << 12) + 1, 8192, P, P, BF, 2, 1, 1, P, P, P, None) == -1
    assert b"split the batch" in lib.lng_last_error()
