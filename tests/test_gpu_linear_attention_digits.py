"""What linear attention's operands keep: scores, states and their gradients enter the matrix products whole (24 bits),
whatever the tensors' type."""

from __future__ import annotations

import pytest
import torch

from ffnmem.memory.linear_attention import linear_attention
from oracle import attention as oa
from oracle.mixing import d as to64

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _whole_numbers(dev, dtype, t, dk, dv, swap, seed):
    """Whole numbers in all tensors.  One column of q and k (swap: of v and dy) is large: its products take 18 bits, odd
    ones among them; so do a few rows (columns) of the states.  Everything else is -1, 0 or 1."""
    gen = torch.Generator().manual_seed(seed)

    def small(*s):
        return torch.randint(-1, 2, s, generator=gen).float() * (torch.rand(*s, generator=gen) < 0.5)

    def odd(bits, *s):
        sign = torch.randint(0, 2, s, generator=gen) * 2 - 1
        return (sign * (2 * torch.randint(1 << (bits - 2), 1 << (bits - 1), s, generator=gen) + 1)).float()

    b, h = 2, 2
    q, k, v, dy = small(b, t, h, dk), small(b, t, h, dk), small(b, t, h, dv), small(b, t, h, dv)
    one, two = (dy, v) if swap else (q, k)
    one[..., 0], two[..., 0] = 4 * odd(8, b, t, h), odd(8, b, t, h)
    state, dend = torch.zeros(b, h, dk, dv), torch.zeros(b, h, dk, dv)
    for s in (state, dend):
        if swap:
            s[..., 1:4] = odd(18, b, h, dk, 3)
        else:
            s[:, :, 1:4] = odd(18, b, h, 3, dv)
    g = torch.zeros(h)
    unit = 2.0 ** -8                                       # keeps results within fp16
    return [x.to(dtype).to(dev) for x in (q, k, v, dy * unit)] + [x.to(dev) for x in (g, state, dend * unit * unit)], unit


@pytest.mark.parametrize("t", [7, 90, 150])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 64), (32, 128), (64, 128), (128, 128)])
@pytest.mark.parametrize("swap", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_whole_numbers_come_out_exactly(dev, dtype, dk, dv, swap, t):
    """Without decays all sums are of whole numbers (times a power of two) below 2^24, which fp32 adds without a rounding in
    any order: a result is the exact one, rounded once."""
    (q, k, v, dy, g, state, dend), unit = _whole_numbers(dev, dtype, t, dk, dv, swap, dk + dv + t)
    leaves = [x.requires_grad_(True) for x in (q, k, v, state)]
    y, end = linear_attention(q, k, v, g, scale=unit, state=state, return_state=True)
    got = [y, end, *torch.autograd.grad([y, end], leaves, [dy, dend])]
    args = dict(q=to64(q), k=to64(k), v=to64(v), g=to64(g), scale=unit, state=to64(state))
    want, mag = [], []
    for out, m in ((want, False), (mag, True)):
        out += oa.linear_attention(mag=m, **args)
        grads = oa.linear_attention_grad(to64(dy), to64(dend), mag=m, **args)
        out += [grads[n] for n in ("q", "k", "v", "state")]
    units = (unit, 1, unit * unit, unit * unit, unit * unit, unit * unit)
    for p, w, m, u, name in zip(got, want, mag, units, ("y", "state", "dq", "dk", "dv", "dstate")):
        assert float(m.max()) / u < 2 ** 24, name          # the premise
        assert torch.equal(p.detach().cpu(), w.float().to(p.dtype)), (name, float((to64(p) - w).abs().max()))
