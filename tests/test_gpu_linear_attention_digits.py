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


def _run(dev, dtype, b, t, h, dk, dv, make, rate, scale=None):
    gen = torch.Generator().manual_seed(t + dk)
    q, k, v, dy = (make(b, t, h, n, generator=gen).to(dtype).to(dev) for n in (dk, dk, dv, dv))
    g = (-rate * torch.rand(b, t, h, generator=gen)).to(dev)
    state, dend = (make(b, h, dk, dv, generator=gen).to(dev) for _ in range(2))
    leaves = [x.requires_grad_(True) for x in (q, k, v, g, state)]
    y, end = linear_attention(q, k, v, g, scale=scale, state=state, return_state=True)
    got = [y, end, *torch.autograd.grad([y, end], leaves, [dy, dend])]
    args = dict(q=to64(q), k=to64(k), v=to64(v), g=to64(g), scale=scale or dk ** -0.5, state=to64(state))
    grads = oa.linear_attention_grad(to64(dy), to64(dend), **args)
    want = [*oa.linear_attention(**args), *(grads[n] for n in ("q", "k", "v", "decay", "state"))]
    return zip(("y", "end", "dq", "dk", "dv", "ddecay", "dstate"), got, want)


LONG = [(2, 333, 4, 64, 64, 0.05), (1, 600, 2, 128, 128, 0.05), (2, 200, 2, 32, 96, 1.0), (3, 31, 2, 40, 72, 0.5)]


@pytest.mark.parametrize("b,t,h,dk,dv,rate", LONG)
def test_fp32_results_are_within_a_few_roundings(dev, b, t, h, dk, dv, rate):
    """Norm by norm: a result's rounding errors are of either sign, so that some hundred additions to it (six products of
    parts for every 32 terms, a step of the state for every chunk) are off by some ten half steps together, and two such
    sums on its way by 2^-24 * 17 = 1e-6.  Operands of two parts, 2^-17 each, would be off by 8e-6."""
    for name, got, want in _run(dev, FP, b, t, h, dk, dv, torch.randn, rate):
        err = float((to64(got) - want).norm() / want.norm())
        assert err <= 1e-6, (name, err)


@pytest.mark.parametrize("b,t,h,dk,dv,rate", LONG)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_16_bit_results_are_fp32_ones_rounded_once(dev, dtype, b, t, h, dk, dv, rate):
    """A value that is off by d before its rounding comes out a step s away from the exact value's rounding with
    probability d / s.  With s <= eps |y| the squares add up to eps * sum(d |y|) <= eps |d| |y|: where the norm error d is
    that of fp32 sums, 1e-6, results are within sqrt(1e-6 eps) of the exactly rounded ones."""
    for name, got, want in _run(dev, dtype, b, t, h, dk, dv, torch.randn, rate):
        if got.dtype == dtype:
            err = float((to64(got) - want.to(dtype).double()).norm() / want.norm())
            assert err <= (1e-6 * torch.finfo(dtype).eps) ** 0.5, (name, err)


@pytest.mark.parametrize("b,t,h,dk,dv", [(2, 32, 4, 64, 64), (2, 33, 4, 32, 32), (1, 300, 2, 128, 128)])
def test_fp32_results_are_off_to_either_side(dev, b, t, h, dk, dv):
    """Values of one sign, no decays, a scale of one.  Sums are rounded to nearest and what is left out of a product is of
    either sign: the mean of thousands of results is that of the exact ones to within less than half of half a step.
    Parts that are cut off leave out 2 * 2^-8 * 2^-16 of a product times the means of two uniform values relative to
    theirs, about 0.7 each: one half step for every product on a result's way."""
    for name, got, want in _run(dev, FP, b, t, h, dk, dv, lambda *s, generator: 1 + torch.rand(*s, generator=generator), 0.0, 1.0):
        off = float(((to64(got) - want) / want).mean()) * 2 ** 24
        assert abs(off) <= 0.4, (name, off)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_the_largest_finite_values_stay_finite(dev, dtype):
    """The type's lowest value among the values, with keys that leave the results in range."""
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randn(1, 90, 2, 32, generator=gen).to(dtype).to(dev) * 2.0 ** -7 for _ in range(2))
    v = torch.full((1, 90, 2, 48), torch.finfo(dtype).min).to(dtype).to(dev)
    g = -0.1 * torch.ones(2, device=dev)
    y, end = linear_attention(q, k, v, g, scale=1.0, return_state=True)
    want = oa.linear_attention(to64(q), to64(k), to64(v), to64(g), 1.0)
    for got, w in zip((y, end), want):
        assert torch.isfinite(got).all()
        err = float(((to64(got) - w) * 2.0 ** -100).norm() / (w * 2.0 ** -100).norm())
        assert err <= (1e-6 if got.dtype == FP else torch.finfo(dtype).eps / 2), err
