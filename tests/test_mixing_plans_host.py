"""What calls of linear attention and group norm ask for, and which they refuse, by their shapes alone."""

from __future__ import annotations

import ctypes

import torch

from lngram_hip import _lib
from lngram_hip.ops import dtype_code

BF, FP = dtype_code(torch.bfloat16), dtype_code(torch.float32)
P = ctypes.c_void_p(4096)


def _attention(b, t, h, **change):
    a = _lib.LinearAttention(B=b, T=t, H=h, Hq=h, Hk=h, Hv=h, K=32, V=32, dtype=BF, token_decay=1, scale=1.0)
    for f in ("q", "k", "v", "decay", "state", "y", "state_out", "checkpoints"):
        setattr(a, f, 4096)
    for n in "qkv":
        for d, size in (("batch", t * h * 32), ("token", h * 32), ("head", 32)):
            setattr(a, f"{n}_{d}", size)
    a.decay_batch, a.decay_token = t * h, h
    for k, v in change.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_distances_of_single_ones_cost_no_copy():
    size = _lib.load().lng_linear_attention_workspace_bytes
    for b, t, h, name in ((1, 64, 4, "batch"), (2, 1, 4, "token"), (2, 64, 1, "head")):
        for n in "qkv":
            assert size(_attention(b, t, h, **{f"{n}_{name}": 3}), 0) == 0, (n, name)
        assert size(_attention(2, 64, 4, **{f"q_{name}": 3}), 0) > 0
