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


def _norm(n, at, c, groups, dtype=BF):
    lib = _lib.load()
    return lib.lng_group_norm(P, dtype, n, at, c, groups, at * c, c, P, P, FP, 1e-5, 1, P, 1 << 50, P, P, P, None)


def _norm_grad(n, at, c, groups, dtype=BF):
    lib = _lib.load()
    return lib.lng_group_norm_grad(P, at * c, c, P, at * c, c, dtype, n, at, c, groups, P, P, FP, 1, P, P, P, 1 << 50, P, P, P, None)


def test_group_norms_of_more_groups_than_a_launch_counts():
    """Sixteen threads a group join its ranges of positions: 2^28 groups are 2^32 threads, where the passes' own launches
    are far from it.  Refused before the first launch."""
    for call in (_norm, _norm_grad):
        for n, at, c, groups in ((1 << 18, 9, 2048, 2048), (1 << 17, 9, 2048, 2048), (1 << 24, 300, 64, 16)):
            assert call(n, at, c, groups) == -1 and b"split the batch" in _lib.load().lng_last_error(), (call, n, at, c, groups)


def test_group_norm_workspaces_go_by_the_groups():
    """A range of positions leaves two numbers a group, and two more a slab of channels, whose ends may share a group: the
    workspace stays below the rows and the statistics that the call reads and writes anyway."""
    size = _lib.load().lng_group_norm_workspace_bytes
    for n, at, c, groups in ((1 << 17, 9, 2048, 2048), (1, 100, 65536, 65536), (1, 100, 65536, 4096), (3, 50, 30000, 10000),
                             (2, 40, 5001, 1667), (1, 5000, 8192, 2048)):
        rows, stats = 2 * n * at * c, 8 * n * groups       # bf16 rows; mean and rstd
        assert 0 < size(n, at, c, groups, 0) <= 2 * rows + stats, (n, at, c, groups)
        assert size(n, at, c, groups, 1) <= 4 * rows + 8 * n * c, (n, at, c, groups)
