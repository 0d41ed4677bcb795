"""Group norm with an activation, channels last, and its backward pass (``lng_group_norm``,
``lng_group_norm_grad``) against the 64-bit form.

Roundings: a thread adds at most 32 values one after the other, joins them with those of the other positions
and channels of its block (at most 256 positions, and 128 channels a lane) and those with up to 256 ranges of
positions, sixteen to a lane: under 450; mean, variance and a sum over both are three such sums on a result's
way, the formula some twenty more.  A weight's gradient adds every position and sample at most."""

from __future__ import annotations

import pytest
import torch

from tests.bounds import within
from ffnmem.memory.norm import GroupNorm, group_norm
from oracle import attention as oa
from oracle.mixing import d as to64

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
K = 3 * 450 + 20


def _make(dev, shape, dtype, wt, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed + sum(shape))
    c = shape[-1]
    x = (torch.randn(*shape, generator=g) + mean * torch.randn(shape[0], *[1] * (len(shape) - 2), c, generator=g)).to(dtype)
    w = b = None
    if wt is not None:
        w, b = (1 + 0.3 * torch.randn(c, generator=g)).to(wt).to(dev), torch.randn(c, generator=g).to(wt).to(dev)
    return x.to(dev), w, b, torch.randn(*shape, generator=g).to(dtype).to(dev)


def _check(x, groups, w, b, dy, silu, eps=1e-5):
    act = "silu" if silu else None
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], eps, act)
    have = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(y, have, dy)))
    assert torch.equal(y.detach(), group_norm(x, groups, w, b, eps, act))          # with and without a graph
    xd, wd, bd, gd = (to64(t) for t in (x, w, b, dy))
    within(y, oa.group_norm(xd, groups, wd, bd, eps, silu), oa.group_norm(xd, groups, wd, bd, eps, silu, mag=True), K, "y")
    want = oa.group_norm_grad(gd, xd, groups, wd, bd, eps, silu)
    mag = oa.group_norm_grad(gd, xd, groups, wd, bd, eps, silu, mag=True)
    rows = x.numel() // x.shape[-1]
    for i, name, k in ((0, "dx", 2 * K), (1, "dw", K + rows), (2, "db", K + rows)):
        if i in grads:
            assert grads[i].dtype == leaves[i].dtype and grads[i].shape == leaves[i].shape
            within(grads[i], want[i], mag[i], k, name)


TOKENS = [((1, 1), 1), ((3, 4), 2), ((5, 14), 7), ((9, 64), 1), ((70, 64), 8), ((33, 1024), 16), ((300, 96), 3),
          ((7, 320), 32), ((5, 2048), 1), ((3, 4096), 2), ((2, 8192), 1), ((3, 2056), 1), ((40, 111), 37), ((3, 8200), 1),
          ((2, 20000), 2), ((6, 5000), 4), ((1500, 40), 20), ((2, 600), 300), ((3, 16384), 2), ((5, 3001), 1)]


@pytest.mark.parametrize("shape,groups", TOKENS)
@pytest.mark.parametrize("dtype,wt", [(BF, BF), (BF, FP), (FP, FP), (HF, HF), (FP, None)])
@pytest.mark.parametrize("silu", [True, False])
def test_one_position_a_sample(dev, shape, groups, dtype, wt, silu):
    x, w, b, dy = _make(dev, shape, dtype, wt)
    if shape[-1] == groups:                    # one value a group: every statistic is that value, dx is zero
        assert torch.equal(group_norm(x, groups, w, b), torch.zeros_like(x) if b is None else b.to(dtype).expand_as(x))
        return
    _check(x, groups, w, b, dy, silu)


SAMPLES = [((2, 3, 4), 2), ((1, 1, 24), 3), ((3, 7, 112), 16), ((4, 40, 320), 32), ((2, 50, 320), 32), ((2, 1500, 64), 8),
           ((1, 4000, 16), 4), ((5, 4, 6, 48), 6), ((2, 3, 5, 7, 10), 5), ((3, 30, 1067), 1), ((2, 9, 2500), 2),
           ((2, 300, 2048), 4), ((1, 700, 4104), 3), ((600, 2, 24), 3), ((2, 11, 33), 11), ((1, 2, 6000), 2),
           ((2, 40, 5001), 3), ((3, 1, 2, 9000), 1)]


@pytest.mark.parametrize("shape,groups", SAMPLES)
@pytest.mark.parametrize("dtype,wt", [(BF, FP), (FP, FP), (HF, HF)])
@pytest.mark.parametrize("silu", [True, False])
def test_whole_samples(dev, shape, groups, dtype, wt, silu):
    _check(*_swap(_make(dev, shape, dtype, wt), groups), silu)


def _swap(made, groups):
    x, w, b, dy = made
    return x, groups, w, b, dy


def test_many_ranges_of_positions(dev):
    """More tiles of positions than ranges: several tiles a block, joined twice."""
    _check(*_swap(_make(dev, (1, 70000, 24), BF, FP), 3), True)
    _check(*_swap(_make(dev, (1, 9000, 512), FP, FP), 8), False)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strided_rows(dev, dtype):
    x, w, b, dy = _make(dev, (4, 30, 64), dtype, FP)
    wide = torch.randn(4, 30, 200, device=dev).to(dtype)
    for v in (wide[..., 8:72], wide[..., 3:67], wide[..., ::2][..., :64], x.transpose(0, 1).contiguous().transpose(0, 1),
              x[:1].expand(4, 30, 64), wide[:, ::3, 64:128]):
        _check(v, 4, w, b, dy[:, :v.shape[1]], True)
        _check(v[:, 0], 4, w, b, dy[:, 0], True)
    _check(x, 4, w, b, dy[:1, :1].expand(4, 30, 64), True)
    x5 = torch.randn(2, 6, 5, 3, 16, device=dev).to(dtype)
    _check(x5.transpose(1, 2), 2, None, None, x5.transpose(1, 2), False)


def test_large_means_and_constant_groups(dev):
    """The variance is formed around the mean: a mean of 2^12 deviations costs 2^12 of x's own steps, no more."""
    for shape, groups in (((50, 64), 2), ((3, 200, 32), 4), ((2, 5000, 32), 4)):
        x, w, b, dy = _make(dev, shape, FP, FP)
        _check(x + 4096, groups, w, b, dy, False)
        flat = torch.full_like(x, 3.25)
        y = group_norm(flat, groups, w, b)
        assert torch.allclose(y, b.expand_as(y), atol=1e-3)


def test_activation_at_its_ends(dev):
    """z from -200 to 200, where silu(z) is 0 or z."""
    x, w, b, dy = _make(dev, (40, 64), FP, FP)
    _check(x, 4, w * 30, b * 100, dy, True)
    _check(x.to(BF), 4, (w * 30).to(BF), (b * 100).to(BF), dy.to(BF), True)
    x, w, b, dy = _make(dev, (2, 300, 32), FP, FP)
    _check(x, 4, w * 30, b * 100, dy, True)


def test_weights_one_by_one(dev):
    for shape in ((20, 48), (3, 20, 48), (2, 900, 48)):
        x, w, b, dy = _make(dev, shape, BF, BF)
        _check(x, 3, w, None, dy, True)
        _check(x, 3, None, b, dy, True)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        ref = torch.autograd.grad(group_norm(leaves[0], 3, leaves[1], leaves[2], activation="silu"), leaves, dy)
        for i in range(3):
            v = [x, w, b]
            v[i] = leaves[i]
            assert torch.equal(torch.autograd.grad(group_norm(v[0], 3, v[1], v[2], activation="silu"), leaves[i], dy)[0], ref[i])


def test_a_sample_does_not_see_the_others(dev):
    for shape in ((6, 96), (6, 9, 96), (6, 900, 96)):
        x, w, b, dy = _make(dev, shape, BF, FP)
        clean = group_norm(x, 3, w, b, activation="silu")
        x[2] = float("nan")
        x[4][..., 0] = float("inf")
        y = group_norm(x, 3, w, b, activation="silu")
        for i in (0, 1, 3, 5):
            assert torch.equal(y[i], clean[i])
        assert torch.isnan(y[2]).all() and torch.equal(y[4][..., 32:], clean[4][..., 32:])


def test_empty(dev):
    w = torch.ones(8, device=dev).requires_grad_(True)
    for shape in ((0, 8), (0, 5, 8), (3, 0, 8)):
        x = torch.zeros(*shape, device=dev, requires_grad=True)
        y = group_norm(x, 2, w, w)
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
        assert gx.shape == shape and (gw == 0).all()


def test_equal_calls_other_stream_and_graph(dev):
    for shape in ((900, 256), (3, 20, 256), (3, 2000, 64)):
        x, w, b, dy = _make(dev, shape, BF, FP)
        x, w, b = (t.requires_grad_(True) for t in (x, w, b))

        def step():
            y = group_norm(x, 8, w, b, activation="silu")
            return [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]

        want = step()
        st = torch.cuda.Stream(dev)
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            got = step()
        torch.cuda.current_stream(dev).wait_stream(st)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for rep in range(3):
            with torch.no_grad():
                x.copy_(torch.randn(*shape, device=dev))
            ref = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, ref)), rep


def test_saved_tensors_that_move(dev):
    """What a graph keeps may come back elsewhere and in another layout (offloaded activations)."""
    wide = torch.randn(3, 40, 200, device=dev)
    for x in (wide[..., 3:67], wide[:, 0, 8:72]):
        _, w, b, dy = _make(dev, tuple(x.shape), FP, FP)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        with torch.autograd.graph.save_on_cpu():
            y = group_norm(leaves[0], 4, leaves[1], leaves[2], activation="silu")
        # rows of another address are read in other pieces and summed in another order: within the bounds of any call
        xd, wd, bd, gd = (to64(t) for t in (x, w, b, dy))
        args = (gd, xd, 4, wd, bd, 1e-5, True)
        for got, want, mag, k in zip(torch.autograd.grad(y, leaves, dy), oa.group_norm_grad(*args),
                                     oa.group_norm_grad(*args, mag=True), (2 * K, K + 120, K + 120)):
            within(got, want, mag, k)


def test_module_and_refusals(dev):
    m = GroupNorm(4, 32, activation="silu").to(dev)
    x = torch.randn(3, 5, 32, device=dev)
    assert torch.equal(m(x), group_norm(x, 4, m.weight, m.bias, activation="silu"))
    assert m(x.to(BF)).dtype == BF and m.to(BF)(x.to(HF)).dtype == HF
    w = torch.ones(32, device=dev)
    for err, call in ((ValueError, lambda: group_norm(x, 5, w, w)), (ValueError, lambda: group_norm(x, 0, w, w)),
                      (ValueError, lambda: group_norm(x, 4, w[:8], w)), (ValueError, lambda: group_norm(x[0, 0], 4, w, w)),
                      (ValueError, lambda: group_norm(x, 4, w, w, activation="gelu")), (ValueError, lambda: m(x[..., :16])),
                      (TypeError, lambda: group_norm(x, 4, w.to(BF), w.to(BF))), (TypeError, lambda: group_norm(x.double(), 4)),
                      (ValueError, lambda: group_norm(x[..., :0], 1)), (RuntimeError, lambda: group_norm(x, 4, w.cpu(), w))):
        with pytest.raises(err):
            call()


def test_positions_past_32_bit_offsets(dev):
    """Rows more than 2^31 elements into one buffer, in both passes."""
    big = torch.empty((1 << 31) + (1 << 26), dtype=BF, device=dev)
    rows = big.as_strided((2, 500, 32), (1 << 31, 1 << 17, 1))
    x, w, b, dy = _make(dev, (2, 500, 32), BF, FP)
    rows.copy_(x)
    assert torch.equal(group_norm(rows, 4, w, b), group_norm(x, 4, w, b))
    tokens = big.as_strided((17, 32), (1 << 27, 1))
    tokens.copy_(x[0, :17])
    assert torch.equal(group_norm(tokens, 4, w, b), group_norm(x[0, :17].contiguous(), 4, w, b))
