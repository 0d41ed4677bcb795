"""Error bounds of fp32 kernels whose outputs are rounded once to their type."""

from __future__ import annotations

import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def within(got: torch.Tensor, want: torch.Tensor, mag: torch.Tensor, k: float, what="") -> None:
    """``|got - want| <= half a step of got's type * |want| + k * 2^-24 * mag``: one rounding to the type, and k
    fp32 roundings, each relative to the size of the sum it happens in (mag).  Below the type's smallest
    normal number a step is absolute."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    f = torch.finfo(got.dtype)
    got = got.detach().to("cpu", torch.float64)
    assert torch.isfinite(got).all(), what
    half = f.eps / 2 if got.dtype != torch.float32 else 0.0
    tol = f.eps / 2 * want.abs() + (1 + half) * (k * U32 + 1e-12) * mag + f.tiny
    over = (got - want).abs() - tol
    assert not over.numel() or float(over.max()) <= 0, (
        what, "worst", float(over.max()), "at", int(over.argmax()), "got", float(got.flatten()[over.argmax()]),
        "want", float(want.flatten()[over.argmax()]), "mag", float((mag + 0 * want).flatten()[over.argmax()]))
