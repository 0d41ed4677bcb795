"""The short causal convolution, its backward pass and its single-token step (``lng_short_conv*``) against
the 64-bit form."""

from __future__ import annotations

import pytest
import torch

from tests.bounds import within
from ffnmem.memory.short_conv import short_conv, short_conv_step
from lngram_hip import ops
from oracle import mixing

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _make(dev, b, t, c, k, dil, dtype, wt=None, hist=True, ragged=False, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * b + t + c)
    wt = wt or dtype

    def r(*s, dt=dtype):
        return torch.randn(*s, generator=g).to(dt).to(dev)

    lengths = None
    if ragged:
        lengths = torch.randint(0, t + 1, (b,), generator=g, dtype=torch.int32)
        lengths[0] = t
        lengths = lengths.to(dev)
    return dict(x=r(b, t, c), w=r(c, k, dt=wt), bias=r(c, dt=wt), dil=dil,
                hist=r(b, (k - 1) * dil, c) if hist else None, lengths=lengths, dy=r(b, t, c), dh=r(b, (k - 1) * dil, c))


def _oracle(s, silu, leaves=()):
    v = {k: mixing.d(s[k]) for k in ("x", "w", "bias", "hist")}
    for k in leaves:
        v[k] = v[k].requires_grad_(True)
    lengths = None if s["lengths"] is None else s["lengths"].cpu()
    return v, mixing.short_conv(v["x"], v["w"], v["bias"], s["dil"], silu, v["hist"], lengths)


def _check(s, silu=True, grads=True):
    """Against the 64-bit form and autograd through it.  Roundings: K + 1 of the taps' sum and a handful of the
    activation's (slope at most 1.1); the gradients add up K such products, the weights' every position."""
    act = "silu" if silu else None
    kw = dict(dilation=s["dil"], activation=act, lengths=s["lengths"], return_history=True)
    y, nxt = short_conv(s["x"], s["w"], s["bias"], history=s["hist"], **kw)
    names = [n for n in ("x", "w", "bias", "hist") if s[n] is not None]
    v, (want, want_h) = _oracle(s, silu, names)
    k = s["w"].shape[1]
    absd = {n: None if t is None else mixing.d(t).abs() for n, t in s.items() if isinstance(t, torch.Tensor) or t is None}
    lengths = None if s["lengths"] is None else s["lengths"].cpu()
    mag, _ = mixing.short_conv(absd["x"], absd["w"], absd["bias"], s["dil"], False, absd["hist"], lengths)
    within(y, want.detach(), mag, 1.1 * (k + 1) + 8, "y")
    assert torch.equal(nxt.double().cpu(), want_h.detach()), "history"
    if not grads:
        return
    leaves = {n: s[n].detach().requires_grad_(True) for n in names}
    y2, nxt2 = short_conv(leaves["x"], leaves["w"], leaves["bias"], history=leaves.get("hist"), **kw)
    assert torch.equal(y2.detach(), y) and torch.equal(nxt2.detach(), nxt)
    got = dict(zip(names, torch.autograd.grad([y2, nxt2], list(leaves.values()), [s["dy"], s["dh"]])))
    dyd, dhd = mixing.d(s["dy"]), mixing.d(s["dh"])
    ref = dict(zip(names, torch.autograd.grad([want, want_h], [v[n] for n in names], [dyd, dhd])))
    # sizes of the sums: |dpre| is at most 1.1 |dy|, its own error that of pre (the slope's slope is at most 0.5)
    amp = dyd.abs() * (1.1 + mag)
    vm = {n: mixing.d(s[n]).abs().requires_grad_(True) for n in names}
    ym, hm = mixing.short_conv(vm["x"], vm["w"], vm["bias"], s["dil"], False, vm.get("hist"), lengths)
    mags = dict(zip(names, torch.autograd.grad([ym, hm], [vm[n] for n in names], [amp, dhd.abs()])))
    steps = s["x"].shape[0] * s["x"].shape[1]
    for n in names:
        assert got[n].dtype == s[n].dtype
        within(got[n], ref[n], mags[n], 3 * k + 20 + (steps if n in ("w", "bias") else 0), "d" + n)


@pytest.mark.parametrize("b,t,c,k,dil", [(1, 1, 8, 4, 1), (2, 1, 5, 2, 1), (3, 2, 64, 4, 3), (2, 17, 64, 4, 1),
                                         (2, 33, 40, 3, 2), (1, 130, 256, 4, 3), (3, 65, 1000, 4, 1), (2, 50, 7, 4, 1),
                                         (2, 40, 24, 5, 2), (2, 19, 16, 8, 1), (2, 9, 16, 1, 1), (1, 6, 32, 4, 7),
                                         (4, 200, 2048, 4, 1), (1, 3000, 512, 2, 1)])
@pytest.mark.parametrize("dtype,wt", [(BF, BF), (BF, FP), (FP, FP), (HF, HF)])
def test_shapes_and_types(dev, b, t, c, k, dil, dtype, wt):
    _check(_make(dev, b, t, c, k, dil, dtype, wt))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_wide_tiles(dev, dtype):
    # so many positions that a thread takes 16 of them, in both directions
    s = _make(dev, 4, 1100, 2048, 4, 1, dtype)
    _check(s)
    _check(dict(s, dil=3, hist=None, dh=torch.zeros(4, 9, 2048, device=dev, dtype=dtype)))


@pytest.mark.parametrize("t,c,k,dil", [(29, 64, 4, 1), (29, 64, 4, 3), (5, 24, 4, 3), (40, 9, 3, 2)])
@pytest.mark.parametrize("silu,hist", [(True, True), (True, False), (False, True)])
def test_ragged_batches(dev, t, c, k, dil, silu, hist):
    s = _make(dev, 7, t, c, k, dil, BF, hist=hist, ragged=True)
    s["lengths"][1], s["lengths"][2], s["lengths"][3] = 0, 1, min(2, t)
    _check(s, silu)


def test_what_stands_behind_a_sequence_is_not_read(dev):
    s = _make(dev, 4, 20, 64, 4, 1, BF, ragged=True)
    s["lengths"].copy_(torch.tensor([20, 7, 0, 13]))
    dirty = dict(s, x=s["x"].clone(), dy=s["dy"].clone())
    for i, n in enumerate((20, 7, 0, 13)):
        dirty["x"][i, n:] = float("nan")
        dirty["dy"][i, n:] = float("inf")
    outs = []
    for v in (s, dirty):
        y, h = ops.short_conv(v["x"], v["w"], v["bias"], 1, True, v["hist"], v["lengths"], True)
        outs.append([y, h, *ops.short_conv_grad(v["dy"], v["x"], v["w"], v["bias"], 1, True, v["hist"], v["lengths"],
                                                v["dh"])])
    assert all(torch.equal(p, q) for p, q in zip(*outs))
    assert (outs[0][0][1, 7:] == 0).all() and (outs[0][2][1, 7:] == 0).all()
    # lengths past the ends are the ends
    far = s["lengths"].clone()
    far[0], far[2] = 1000, -5
    y, _ = ops.short_conv(s["x"], s["w"], s["bias"], 1, True, s["hist"], far, True)
    assert torch.equal(y, outs[0][0])


def test_infinite_rows_reach_their_window_only(dev):
    for k in (3, 5):                                                  # 5: registers of absent taps
        s = _make(dev, 1, 24, 16, k, 2, FP, hist=False)
        s["x"][0, 10] = float("inf")
        y = short_conv(s["x"], s["w"], s["bias"], dilation=2, activation=None)
        reach = [10 + 2 * j for j in range(k) if 10 + 2 * j < 24]
        bad = ~torch.isfinite(y[0]).all(-1).cpu()
        assert bad.nonzero().flatten().tolist() == reach


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strided_rows(dev, dtype):
    s = _make(dev, 3, 21, 64, 4, 1, dtype)
    wide = torch.randn(3, 21, 200, device=dev).to(dtype)
    for x in (wide[..., :64], wide[..., 64:128], wide[..., 3:67], wide[:, ::3, 8:72], wide.transpose(0, 1)[:3, :, :64],
              wide[:1, :, :64].expand(3, 21, 64), wide[..., ::2][..., :64]):
        v = dict(s, x=x, dy=s["dy"][:, :x.shape[1]])
        _check(v if x.shape[1] == 21 else dict(v, lengths=None))


def test_in_parts_equals_the_whole(dev):
    s = _make(dev, 2, 60, 64, 4, 3, BF)
    whole, end = short_conv(s["x"], s["w"], s["bias"], dilation=3, history=s["hist"], return_history=True)
    h, parts = s["hist"], []
    for a, b in ((0, 7), (7, 8), (8, 40), (40, 60)):
        y, h = short_conv(s["x"][:, a:b], s["w"], s["bias"], dilation=3, history=h, return_history=True)
        parts.append(y)
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(h, end)
    h2, steps = s["hist"].clone(), []
    for i in range(60):
        steps.append(short_conv_step(s["x"][:, i], h2, s["w"], s["bias"], dilation=3))
    assert torch.equal(torch.stack(steps, 1), whole) and torch.equal(h2, end)


@pytest.mark.parametrize("b,c,k,dil", [(1, 8, 4, 1), (8, 1024, 4, 1), (5, 37, 3, 2), (64, 256, 4, 3), (3, 16, 1, 1), (2, 24, 8, 2)])
@pytest.mark.parametrize("dtype,wt", [(BF, BF), (BF, FP), (FP, FP), (HF, HF)])
def test_step(dev, b, c, k, dil, dtype, wt):
    s = _make(dev, b, 1, c, k, dil, dtype, wt)
    want, nxt = ops.short_conv(s["x"], s["w"], s["bias"], dil, True, s["hist"], None, True)
    h, out = s["hist"].clone(), torch.full_like(s["hist"], 7)
    y = short_conv_step(s["x"][:, 0], h, s["w"], s["bias"], dil, out_history=out)
    assert torch.equal(h, s["hist"]) and torch.equal(out, nxt) and torch.equal(y, want[:, 0])
    wide = torch.randn(b, 3 * c, device=dev).to(dtype)
    x = wide[:, c:2 * c]
    y = short_conv_step(x, h, s["w"], s["bias"], dil)                 # in place, a part of wider rows
    want, nxt = ops.short_conv(x[:, None], s["w"], s["bias"], dil, True, s["hist"], None, True)
    assert torch.equal(y, want[:, 0]) and torch.equal(h, nxt)


@pytest.mark.parametrize("k,dil", [(2, 1), (3, 2), (4, 3), (5, 1)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_wide_tiles_of_odd_channels(dev, k, dil, dtype):
    """Enough positions for the longest tiles, channel by channel, with a history and ragged ends."""
    _check(_make(dev, 3, 1500, 501, k, dil, dtype, ragged=True), True)


def test_step_in_place_is_seen_by_a_graph_that_kept_the_history(dev):
    s = _make(dev, 2, 4, 16, 4, 1, FP)
    w = s["w"].detach().requires_grad_(True)
    y = short_conv(s["x"], w, s["bias"], history=s["hist"])
    short_conv_step(s["x"][:, 0], s["hist"], s["w"], s["bias"])
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


def test_empty_batches(dev):
    s = _make(dev, 2, 4, 16, 4, 1, BF)
    y, h = short_conv(s["x"][:, :0], s["w"], s["bias"], history=s["hist"], return_history=True)
    assert y.shape == (2, 0, 16) and torch.equal(h, s["hist"])
    y, h = short_conv(s["x"][:0], s["w"], s["bias"], return_history=True)
    assert y.shape == (0, 4, 16) and h.shape == (0, 3, 16)
    for x, hist, dy, dh in ((s["x"][:, :0], s["hist"], s["dy"][:, :0], s["dh"]), (s["x"][:0], None, s["dy"][:0], None)):
        dx, dw, db, dhist = ops.short_conv_grad(dy, x, s["w"], s["bias"], 1, True, hist, None, dh)
        assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
        if dh is not None:
            assert torch.equal(dhist, dh)
    assert short_conv_step(s["x"][:0, 0], s["hist"][:0], s["w"]).shape == (0, 16)


def test_equal_calls_give_equal_bits(dev):
    s = _make(dev, 4, 700, 256, 4, 1, BF)
    a = [ops.short_conv_grad(s["dy"], s["x"], s["w"], s["bias"], 1, True, s["hist"], None, s["dh"]) for _ in range(3)]
    assert all(torch.equal(p, q) for other in a[1:] for p, q in zip(a[0], other))


def test_graph_replays(dev):
    s = _make(dev, 2, 100, 64, 4, 1, BF)
    leaves = [s[n].requires_grad_(True) for n in ("x", "w", "bias", "hist")]

    def step():
        y, h = short_conv(leaves[0], leaves[1], leaves[2], history=leaves[3], return_history=True)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], leaves, [s["dy"], s["dh"]])]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(2, 100, 64, device=dev))
        ref = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref)), rep


def test_refusals(dev):
    s = _make(dev, 2, 6, 16, 4, 1, BF)
    x, w, b, h = s["x"], s["w"], s["bias"], s["hist"]
    for err, kw in ((ValueError, dict(x=x[0])), (ValueError, dict(weight=w[:8])), (ValueError, dict(bias=b[:8])),
                    (TypeError, dict(x=x.double())), (TypeError, dict(weight=w.to(HF), bias=None)),
                    (TypeError, dict(weight=w.float())), (ValueError, dict(history=h[:, :2])),
                    (TypeError, dict(history=h.float())), (ValueError, dict(dilation=0)), (ValueError, dict(dilation=2, history=h)),
                    (ValueError, dict(activation="relu")), (ValueError, dict(weight=torch.randn(16, 9, device=dev).to(BF))),
                    (ValueError, dict(lengths=torch.zeros(3, dtype=torch.int32, device=dev))),
                    (TypeError, dict(lengths=torch.zeros(2, device=dev))), (RuntimeError, dict(bias=b.cpu()))):
        with pytest.raises(err):
            short_conv(**{**dict(x=x, weight=w, bias=b), **kw})
    with pytest.raises(RuntimeError, match="no_grad"):
        short_conv_step(x[:, 0], h, w.clone().requires_grad_(True), b)
    with pytest.raises(ValueError, match="contiguous"):
        short_conv_step(x[:, 0], h.transpose(0, 1).contiguous().transpose(0, 1), w, b)
    both = torch.zeros(3, 3, 16, device=dev, dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        short_conv_step(x[:, 0], both[:2], w, b, out_history=both[1:])


def test_long_dilations_and_lengths_past_32_bits(dev):
    for t in (1, 3, 40):
        _check(_make(dev, 2, t, 24, 4, 50, BF))                       # fewer positions than residue classes
    s = _make(dev, 3, 9, 16, 4, 1, BF)
    far = torch.tensor([2 ** 32 + 2, 4, -2 ** 33], device=dev)        # the first is past the end, not 2
    y = short_conv(s["x"], s["w"], s["bias"], history=s["hist"], lengths=far)
    assert torch.equal(y, short_conv(s["x"], s["w"], s["bias"], history=s["hist"],
                                     lengths=torch.tensor([9, 4, 0], dtype=torch.int32, device=dev)))
