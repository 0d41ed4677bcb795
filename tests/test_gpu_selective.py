"""The selective scan, its backward pass and its single-token step (``lng_selective_*``) against the 64-bit
form.

Roundings of the scan: a state is a product of decays, and every token multiplies it by an exponential whose
argument s * A carries some 8 half steps (the softplus, the product, log2 e) relative to |s A| and the
result two; one more each for the product and the sum.  |x| exp(-|x|) is below 1, so the arguments' errors
of all tokens together stay below 8 half steps of the state's size, and the others add up to 4 a token: 4 T
+ 40 with the input's and the output's own steps.  The gradients run over T tokens once more, in both
directions, and a sum over tokens, sequences or channels adds its length."""

from __future__ import annotations

import pytest
import torch

from tests.bounds import within
from ffnmem.memory.selective import selective_scan, selective_step
from lngram_hip import ops
from oracle import mixing

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
LEAVES = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")


def _make(dev, b, t, c, n, g=1, dtype=FP, gate=True, start=True, ragged=False, plain=False, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * t + c + n)

    def r(*s, dt=dtype, std=1.0):
        return (torch.randn(*s, generator=gen) * std).to(dt).to(dev)

    lengths = None
    if ragged:
        lengths = torch.randint(0, t + 1, (b,), generator=gen, dtype=torch.int32)
        lengths[0] = t
        lengths = lengths.to(dev)
    step = torch.exp(torch.empty(c).uniform_(-6.9, -2.3, generator=gen))
    s = dict(u=r(b, t, c), dt=r(b, t, c, std=0.5), A=-(0.5 + 2 * torch.rand(c, n, generator=gen)).to(dev) * n ** 0.5,
             B=r(b, t, g, n), C=r(b, t, g, n), D=r(c, dt=FP), z=r(b, t, c) if gate else None,
             dt_bias=torch.log(torch.expm1(step)).to(dev), state=r(b, c, n, dt=FP) if start else None,
             lengths=lengths, dy=r(b, t, c), dend=r(b, c, n, dt=FP), soft=True)
    if plain:                                                        # steps as they come, no bias, no skip
        s.update(dt=(0.2 * torch.rand(b, t, c, generator=gen)).to(dtype).to(dev), dt_bias=None, D=None, soft=False)
    return s


def _call(s, leaves=None, want_state=True):
    v = {**{k: s[k] for k in LEAVES}, **(leaves or {})}
    return selective_scan(v["u"], v["dt"], v["A"], v["B"], v["C"], D=v["D"], z=v["z"], dt_bias=v["dt_bias"],
                          dt_softplus=s["soft"], state=v["state"], lengths=s["lengths"], return_state=want_state)


def _check(s, grads=True):
    b, t, c = s["u"].shape
    y, end = _call(s)
    v = {k: mixing.d(s[k]) for k in LEAVES}
    for k in ("B", "C"):
        if v[k].dim() == 3:
            v[k] = v[k].unsqueeze(2)
    kw = dict(softplus=s["soft"], lengths=None if s["lengths"] is None else s["lengths"].cpu(), **v)
    (wy, wend), (my, mend) = mixing.selective_scan(**kw), mixing.selective_scan(mag=True, **kw)
    within(y, wy, my, 4 * t + 40, "y")
    within(end, wend, mend, 4 * t + 40, "state")
    if not grads:
        return
    names = [k for k in LEAVES if s[k] is not None]
    leaves = {k: s[k].detach().requires_grad_(True) for k in names}
    y2, end2 = _call(s, leaves)
    assert torch.equal(y2.detach(), y) and torch.equal(end2.detach(), end)
    got = dict(zip(names, torch.autograd.grad([y2, end2], list(leaves.values()), [s["dy"], s["dend"]])))
    dy, dend = mixing.d(s["dy"]), mixing.d(s["dend"])
    want, mag = mixing.selective_grad(dy, dend, **kw), mixing.selective_grad(dy, dend, mag=True, **kw)
    n = s["A"].shape[1]
    sums = {"B": c, "C": c, "A": b * t, "D": b * t, "dt_bias": b * t, "u": n, "dt": n, "z": n, "state": 0}
    for k in names:
        assert got[k].dtype == s[k].dtype
        within(got[k], want[k].reshape(got[k].shape), mag[k].reshape(got[k].shape), 8 * t + 80 + sums[k], "d" + k)


@pytest.mark.parametrize("b,t,c,n,g", [(1, 1, 1, 1, 1), (2, 3, 5, 4, 1), (1, 16, 64, 16, 1), (2, 17, 65, 16, 1),
                                       (3, 33, 24, 12, 2), (1, 70, 300, 16, 4), (2, 40, 130, 5, 1), (1, 31, 64, 64, 1),
                                       (1, 20, 70, 100, 1), (1, 18, 16, 256, 1), (2, 64, 8, 16, 8)])
@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_shapes_and_types(dev, b, t, c, n, g, dtype):
    _check(_make(dev, b, t, c, n, g, dtype))


@pytest.mark.parametrize("b,t,c", [(1, 64, 64), (1, 65, 100), (2, 130, 64), (1, 400, 192), (3, 257, 64)])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_several_chunks(dev, b, t, c, dtype):
    _check(_make(dev, b, t, c, 16, 1, dtype))


@pytest.mark.parametrize("b,t,c,n,g", [(1, 600, 70, 16, 1), (2, 1030, 24, 20, 2), (1, 513, 64, 12, 1),
                                       (2, 512, 40, 9, 1), (3, 100, 33, 17, 3), (2, 48, 60, 32, 1), (1, 37, 1, 33, 1),
                                       (3, 530, 700, 16, 1), (2, 15, 6, 24, 2), (1, 300, 130, 5, 1), (2, 257, 9, 1, 1),
                                       (2, 256, 20, 8, 4), (2, 1000, 30, 50, 1), (1, 1025, 20, 64, 1),
                                       (3, 90, 33, 33, 3), (1, 1024, 8, 48, 2), (2, 33, 70, 64, 1), (1, 50, 12, 65, 1)])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_states_over_lanes_and_over_time(dev, b, t, c, n, g, dtype):
    """Both ways to run a prompt, on each side of their rule in lengths, channels and states."""
    _check(_make(dev, b, t, c, n, g, dtype, ragged=b > 1))


@pytest.mark.parametrize("n", [5, 9, 12, 16, 20, 32, 40, 60, 70])
@pytest.mark.parametrize("t", [20, 600])
def test_infinite_input_stays_infinite(dev, n, t):
    """Positive B and C: what follows an infinite input is infinite in its channel and finite in the others, and
    nothing multiplies it by a state that isn't there."""
    s = _make(dev, 1, t, 9, n, gate=False, plain=True, start=False)
    s["u"] = s["u"].abs()
    s["u"][0, 7, 4] = float("inf")
    s["B"], s["C"] = s["B"].abs() + 0.1, s["C"].abs() + 0.1
    s["dt"] = s["dt"] * 0.01 + 1e-3                                  # decays far from zero over all of the tokens
    y, end = _call(s)
    assert torch.isinf(y[0, 7:, 4]).all() and (y[0, 7:, 4] > 0).all() and torch.isinf(end[0, 4]).all()
    rest = [i for i in range(9) if i != 4]
    assert torch.isfinite(y[:, :, rest]).all() and torch.isfinite(y[0, :7]).all()


@pytest.mark.parametrize("t", [5, 48, 150, 260])
@pytest.mark.parametrize("start", [True, False])
def test_ragged_batches(dev, t, start):
    s = _make(dev, 6, t, 72, 8, 2, BF, start=start, ragged=True)
    s["lengths"][1], s["lengths"][2], s["lengths"][3] = 0, 1, t - 1
    _check(s)


def test_without_gate_bias_or_skip(dev):
    _check(_make(dev, 2, 90, 80, 16, gate=False, plain=True, start=False))
    s = _make(dev, 2, 90, 80, 16, dtype=BF)
    _check(dict(s, B=s["B"][:, :, 0], C=s["C"][:, :, 0]))              # one group without its dimension


def test_steps_of_all_sizes(dev):
    """The softplus from -30 to 30, and decays from none to all."""
    s = _make(dev, 2, 40, 64, 8)
    s["dt"].copy_(torch.linspace(-30, 30, s["dt"].numel(), device=dev).view(64, 2, 40).permute(1, 2, 0))
    s["dt_bias"].zero_()
    _check(s)
    s["A"].zero_()                                                     # a plain sum
    s["dt"].clamp_(max=1)
    _check(s)


def test_what_stands_behind_a_sequence_is_not_read(dev):
    for t in (24, 200):
        s = _make(dev, 4, t, 70, 16, ragged=True, dtype=BF)
        own = (t, 7, 0, t // 2 + 1)
        s["lengths"].copy_(torch.tensor(own))
        dirty = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        for i, n in enumerate(own):
            for k in ("u", "dt", "B", "C", "z", "dy"):
                dirty[k][i, n:] = float("nan")
        outs = []
        for v in (s, dirty):
            leaves = {k: v[k].requires_grad_(True) for k in LEAVES}
            y, end = _call(v, leaves)
            outs.append([y.detach(), end.detach(), *torch.autograd.grad([y, end], list(leaves.values()),
                                                                       [v["dy"], v["dend"]])])
        for p, q, k in zip(*outs, ("y", "end", *LEAVES)):
            assert torch.equal(p, q), k
        assert (outs[0][0][1, 7:] == 0).all() and torch.equal(outs[0][1][2], s["state"][2])


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strided_inputs(dev, dtype):
    s = _make(dev, 2, 50, 64, 16, 1, dtype)
    wide = torch.randn(2, 50, 400, device=dev).to(dtype)
    low = torch.randn(2, 50, 5 + 32, device=dev).to(dtype)             # B and C behind an odd number of columns
    v = dict(s, u=wide[..., :64], z=wide[..., 101:165], B=low[..., 5:21], C=low[..., 21:])
    _check(v)
    _check(dict(s, u=wide[..., ::2][..., :64], dt=s["dt"].transpose(0, 1).contiguous().transpose(0, 1),
                B=s["B"][:, :1].expand(2, 50, 1, 16), dy=s["dy"][:1].expand(2, 50, 64)))


def test_in_parts_equals_the_whole(dev):
    """A prompt in two parts and then token by token: the states that come back continue the sequence."""
    s = _make(dev, 3, 60, 40, 16, 2, BF)
    kw = dict(D=s["D"], dt_bias=s["dt_bias"], dt_softplus=True)
    whole, end = _call(s)
    st, ys = s["state"], []
    for a, b in ((0, 16), (16, 37)):
        cut = [s[k][:, a:b] for k in ("u", "dt", "B", "C", "z")]
        y, st = selective_scan(cut[0], cut[1], s["A"], cut[2], cut[3], z=cut[4], state=st, return_state=True, **kw)
        ys.append(y)
    for i in range(37, 60):
        nxt = torch.empty_like(st)
        cut = [s[k][:, i] for k in ("u", "dt", "B", "C", "z")]
        before = st.clone()
        ys.append(selective_step(st, cut[0], cut[1], s["A"], cut[2], cut[3], z=cut[4], out_state=nxt, **kw)[:, None])
        assert torch.equal(st, before)
        st = nxt
    v = {k: mixing.d(s[k]) for k in LEAVES}
    my, mend = mixing.selective_scan(softplus=True, mag=True, **v)
    # both are within the bound of the exact values, y after a rounding to bf16 each
    k = 2 * (4 * 60 + 40)
    within(st, mixing.d(end), mend, k, "state")
    within(torch.cat(ys, 1), mixing.d(whole), my + 1.02 * 2.0 ** 16 / k * mixing.d(whole).abs(), k, "y")


@pytest.mark.parametrize("b,c,n,g", [(1, 1, 1, 1), (8, 1024, 16, 1), (5, 37, 6, 1), (3, 40, 12, 4), (2, 70, 64, 1),
                                     (2, 9, 200, 1), (64, 256, 16, 2), (3, 33, 5, 3), (2, 8, 2, 1)])
@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_step(dev, b, c, n, g, dtype):
    s = _make(dev, b, 1, c, n, g, dtype)
    v = {k: mixing.d(s[k]) for k in LEAVES}
    (wy, wend), (my, mend) = (mixing.selective_scan(softplus=True, mag=m, **v) for m in (False, True))
    cut = [s[k][:, 0] for k in ("u", "dt", "B", "C", "z")]
    kw = dict(D=s["D"], z=cut[4], dt_bias=s["dt_bias"], dt_softplus=True)
    st, out = s["state"].clone(), torch.full_like(s["state"], 9)
    y = selective_step(st, cut[0], cut[1], s["A"], cut[2], cut[3], out_state=out, **kw)
    assert torch.equal(st, s["state"])
    within(y, wy[:, 0], my[:, 0], 44 + n, "y")
    within(out, wend, mend, 44, "state")
    y2 = selective_step(st, cut[0], cut[1], s["A"], cut[2], cut[3], **kw)
    assert torch.equal(y2, y) and torch.equal(st, out)                 # in place
    plain = selective_step(s["state"].clone(), cut[0], cut[1].abs(), s["A"], cut[2], cut[3])
    v.update(dt=v["dt"].abs(), D=None, z=None, dt_bias=None)
    (wy, _), (my, _) = (mixing.selective_scan(softplus=False, mag=m, **v) for m in (False, True))
    within(plain, wy[:, 0], my[:, 0], 44 + n, "plain")


def test_step_in_place_is_seen_by_a_graph_that_kept_the_state(dev):
    s = _make(dev, 2, 4, 16, 4)
    A = s["A"].detach().requires_grad_(True)
    y = selective_scan(s["u"], s["dt"], A, s["B"], s["C"], state=s["state"])
    selective_step(s["state"], s["u"][:, 0], s["dt"][:, 0], s["A"], s["B"][:, 0], s["C"][:, 0])
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


def test_step_of_strided_rows(dev):
    s = _make(dev, 4, 1, 24, 16, 1, BF)
    wide = torch.randn(4, 100, device=dev).to(BF)
    u, z, B, C = wide[:, :24], wide[:, 24:48], wide[:, 49:65], wide[:, 65:81]
    a, b = s["state"].clone(), s["state"].clone()
    y1 = selective_step(a, u, s["dt"][:, 0], s["A"], B, C, z=z)
    y2 = selective_step(b, u.contiguous(), s["dt"][:, 0], s["A"], B.contiguous(), C.contiguous(), z=z.contiguous())
    assert torch.equal(y1, y2) and torch.equal(a, b)


def test_empty_batches(dev):
    s = _make(dev, 2, 4, 16, 8, dtype=BF)
    none = {k: s[k][:, :0] for k in ("u", "dt", "B", "C", "z", "dy")}
    v = dict(s, **none)
    leaves = {k: v[k].detach().requires_grad_(True) for k in LEAVES}
    y, end = _call(v, leaves)
    assert y.shape == (2, 0, 16) and torch.equal(end.detach(), s["state"])
    g = dict(zip(LEAVES, torch.autograd.grad([y, end], list(leaves.values()), [v["dy"], s["dend"]])))
    assert torch.equal(g["state"], s["dend"]) and (g["A"] == 0).all() and (g["D"] == 0).all()
    zero = {k: s[k][:0] for k in ("u", "dt", "B", "C", "z", "dy")}
    y, end = _call(dict(s, **zero, state=None))
    assert y.shape == (0, 4, 16) and end.shape == (0, 16, 8)


def test_only_some_gradients(dev):
    s = _make(dev, 2, 30, 32, 16, dtype=BF, start=False)
    full = {k: s[k].detach().requires_grad_(True) for k in LEAVES if s[k] is not None}
    ref = dict(zip(full, torch.autograd.grad(_call(s, full, want_state=False), list(full.values()), s["dy"])))
    for k in ("u", "A", "z"):
        one = {k: s[k].detach().requires_grad_(True)}
        assert torch.equal(torch.autograd.grad(_call(s, one, want_state=False), one[k], s["dy"])[0], ref[k])
    # the final state's gradient alone
    leaf = s["u"].detach().requires_grad_(True)
    _, end = _call(s, {"u": leaf})
    got = torch.autograd.grad(end, leaf, s["dend"])[0]
    want = ops.selective_scan_grad(torch.zeros_like(s["dy"]), s["dend"], ops.selective_scan(
        s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], True, want_checkpoints=True)[2], s["u"], s["dt"],
        s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], True, None, None)["u"]
    assert torch.equal(got, want)


def test_equal_calls_give_equal_bits(dev):
    s = _make(dev, 2, 300, 300, 16, dtype=BF)
    runs = []
    for _ in range(3):
        leaves = {k: s[k].detach().requires_grad_(True) for k in LEAVES}
        y, end = _call(s, leaves)
        runs.append([y, end, *torch.autograd.grad([y, end], list(leaves.values()), [s["dy"], s["dend"]])])
    assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(runs[0], r))


def test_other_stream_and_graph(dev):
    s = _make(dev, 2, 150, 72, 16, dtype=BF)
    want = _call(s)
    st = torch.cuda.Stream(dev)
    st.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(st):
        got = _call(s)
    torch.cuda.current_stream(dev).wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    leaves = {k: s[k].requires_grad_(True) for k in LEAVES}

    def step():
        y, end = _call(s, leaves)
        return [y.detach(), end.detach(), *torch.autograd.grad([y, end], list(leaves.values()), [s["dy"], s["dend"]])]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        with torch.no_grad():
            leaves["u"].copy_(torch.randn(2, 150, 72, device=dev))
        ref = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref)), rep


def test_refusals(dev):
    s = _make(dev, 2, 6, 16, 4, 1, BF)
    for err, kw in ((ValueError, dict(u=s["u"][0])), (ValueError, dict(dt=s["dt"][:, :5])), (TypeError, dict(dt=s["dt"].float())),
                    (ValueError, dict(A=s["A"][:8])), (ValueError, dict(B=s["B"].expand(2, 6, 3, 4), C=s["C"].expand(2, 6, 3, 4))),
                    (ValueError, dict(C=s["C"][..., :3])), (ValueError, dict(D=s["D"][:3])), (ValueError, dict(z=s["z"][:1])),
                    (ValueError, dict(state=s["state"][..., :3])), (TypeError, dict(z=s["z"].to(HF))),
                    (ValueError, dict(A=torch.zeros(16, 257, device=dev), B=torch.zeros(2, 6, 257, device=dev, dtype=BF),
                                      C=torch.zeros(2, 6, 257, device=dev, dtype=BF))),
                    (RuntimeError, dict(A=s["A"].cpu()))):
        v = {**s, **kw}
        with pytest.raises(err):
            _call({**v, "state": v["state"] if "state" in kw else None})
    with pytest.raises(ValueError, match="lengths"):
        _call(dict(s, lengths=torch.ones(3, dtype=torch.int32, device=dev)))
    with pytest.raises(TypeError, match="lengths"):
        _call(dict(s, lengths=torch.ones(2, device=dev)))
    cut = [s[k][:, 0] for k in ("u", "dt", "B", "C")]
    st = s["state"]
    with pytest.raises(RuntimeError, match="no_grad"):
        selective_step(st, cut[0], cut[1], s["A"].clone().requires_grad_(True), cut[2], cut[3])
    with pytest.raises(ValueError, match="contiguous"):
        selective_step(st.transpose(1, 2).contiguous().transpose(1, 2), cut[0], cut[1], s["A"], cut[2], cut[3])
    with pytest.raises(TypeError, match="float32"):
        selective_step(st.to(BF), cut[0], cut[1], s["A"], cut[2], cut[3], out_state=torch.empty_like(st))
    both = torch.zeros(3, 16, 4, device=dev)
    with pytest.raises(ValueError, match="overlaps"):
        selective_step(both[:2], cut[0], cut[1], s["A"], cut[2], cut[3], out_state=both[1:])


def test_lengths_past_32_bits(dev):
    s = _make(dev, 3, 9, 16, 4)
    outs = [_call(dict(s, lengths=v)) for v in (torch.tensor([2 ** 32 + 2, 4, -2 ** 33], device=dev),
                                                torch.tensor([9, 4, 0], dtype=torch.int32, device=dev))]
    assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_rows_far_apart(dev):
    """Sequences that lie token by token in a large buffer, and rows that overlap."""
    s = _make(dev, 2, 40, 64, 16, dtype=BF)
    big = torch.randn(40, 2, 64 * 300, device=dev).to(BF)
    _check(dict(s, u=big.transpose(0, 1)[..., 128:192], dt=s["dt"].as_strided((2, 40, 64), (3, 5, 1))))
