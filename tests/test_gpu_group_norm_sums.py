"""Sums of group norm's backward pass over many positions of one thread."""

from __future__ import annotations

import pytest
import torch

from lngram_hip import ops

pytestmark = pytest.mark.gpu


def test_long_samples_of_a_full_card(dev):
    """Samples enough that each position range is a whole sample, and rows that leave a thread one channel: it adds all 4096
    positions.  Rows of +1 and -1 in equal number and a constant gradient c: h = c, mean(h) = c, mean(h xn) = 0, dx = 0.
    32 positions and 128 such sums one after the other, then 254 channels of 16 lanes, four exchanges and a product by 1 / n:
    under 190 roundings; the bound is 450.  One after the other the 4096 additions of c are rounded the same way for as
    long as the sum stays in a binade: with half a step lost in each of the last 1400 they are off by some 850."""
    n, at, c = 2048, 4096, 254
    x = torch.cat((torch.ones(c // 2), -torch.ones(c // 2))).to(dev).expand(n, at, c)
    const = 1.5 + 0.49 * 2.0 ** -11                     # the step of sums from 2^12 on is 2^-11
    dy = torch.full((c,), const, device=dev).expand(n, at, c)
    stats = torch.stack((torch.zeros(n, 1), torch.ones(n, 1))).to(dev)
    dx = ops.group_norm_grad(dy, x, 1, None, None, False, stats, (True, False, False))[0]
    worst = max(float(part.abs().max()) for part in dx)
    assert worst <= 450 * 2.0 ** -24 * const, worst / const * 2 ** 24
