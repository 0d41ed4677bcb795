"""Calls of linear attention that its documentation allows and whose layouts are unusual."""

from __future__ import annotations

import pytest
import torch

from ffnmem.memory.linear_attention import linear_attention

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("b,t,h", [(1, 1, 1), (2, 1, 1), (1, 5, 1), (1, 1, 3), (1, 70, 2), (3, 4, 2)])
def test_results_that_are_part_of_wider_rows(dev, dtype, b, t, h):
    """The gradient of a concatenation is a slice: where there is one sequence, token or head, its distance to the next is
    any number, and torch counts the slice as contiguous all the same."""
    gen = torch.Generator().manual_seed(b + 10 * t + 100 * h)
    leaves = [torch.randn(b, t, h, 8, generator=gen).to(dtype).to(dev).requires_grad_(True) for _ in range(3)]
    g = (-torch.rand(b, t, h, generator=gen)).to(dev).requires_grad_(True)
    more = torch.randn(b, t, h, 3, generator=gen).to(dtype).to(dev)
    dy = torch.randn(b, t, h, 11, generator=gen).to(dtype).to(dev)
    y = linear_attention(*leaves, g)
    want = torch.autograd.grad(y, [*leaves, g], dy[..., :8].contiguous().clone())
    got = torch.autograd.grad(torch.cat([linear_attention(*leaves, g), more], -1), [*leaves, g], dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_single_sequences_tokens_and_heads_of_any_distance(dev):
    """Inputs as slices of wider rows, one sequence, token or head of them."""
    for b, t, h in ((1, 1, 1), (1, 40, 1), (4, 1, 1)):
        wide = torch.randn(b, t, h, 37, device=dev).to(BF)
        parts = [wide[..., i:i + 8] for i in (0, 8, 16)]
        g = -torch.rand(b, t, h, device=dev)
        assert torch.equal(linear_attention(*parts, g), linear_attention(*(x.contiguous().clone() for x in parts), g))
