"""Linear attention with a decay per head, its backward pass and its single-token step
(``lng_linear_attention_*``) against the 64-bit form.

Roundings.  A sum runs over at most T tokens, K keys and a chunk's 64 tokens once more, in up to six parts each:
6 (T + K + 64).  A weight 2^-d has its exponent's error, 2 |d| 2^-24 ln 2 of itself; the decays of all tokens
together reach at most 2^-126 before they count as zero: 200 half steps, and a few a chunk.  Weights and states
enter the products of a 16-bit type as two bf16 parts, 2^-18 of themselves, 64 half steps each, and as much
again for the product of two second parts: 256; as three parts in fp32: 8.  A gradient goes through two such
sums, in both directions, and a shared head or a decay of all tokens adds its number of terms."""

from __future__ import annotations

import pytest
import torch

from tests.bounds import within
from ffnmem.memory.linear_attention import linear_attention, linear_attention_step
from lngram_hip import ops
from oracle import attention as oa
from oracle.mixing import d as to64

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
LEAVES = ("q", "k", "v", "decay", "state")


def _k(s) -> float:
    t, keys = s["q"].shape[1], s["q"].shape[-1]
    return 6 * (t + keys + 64) + 200 + t / 4 + (8 if s["q"].dtype == FP else 256)


def _make(dev, b, t, h, dk, dv, hq=None, hk=None, hv=None, dtype=FP, token=True, start=True, ragged=False, seed=0, rate=0.5):
    gen = torch.Generator().manual_seed(seed + 7 * t + dk + 3 * dv + h)

    def r(*s, dt=dtype, std=1.0):
        return (torch.randn(*s, generator=gen) * std).to(dt).to(dev)

    lengths = None
    if ragged:
        lengths = torch.randint(0, t + 1, (b,), generator=gen, dtype=torch.int32)
        lengths[0] = t
        lengths = lengths.to(dev)
    decay = (-rate * torch.rand(*((b, t, h) if token else (h,)), generator=gen)).to(dev)
    return dict(q=r(b, t, hq or h, dk), k=r(b, t, hk or h, dk), v=r(b, t, hv or h, dv), decay=decay,
                state=r(b, h, dk, dv, dt=FP) if start else None, lengths=lengths, dy=r(b, t, h, dv),
                dend=r(b, h, dk, dv, dt=FP), scale=None)


def _call(s, leaves=None, want_state=True):
    v = {**{k: s[k] for k in LEAVES}, **(leaves or {})}
    return linear_attention(v["q"], v["k"], v["v"], v["decay"], scale=s["scale"], state=v["state"], lengths=s["lengths"],
                            return_state=want_state)


def _exact(s) -> dict:
    return dict(q=to64(s["q"]), k=to64(s["k"]), v=to64(s["v"]), g=to64(s["decay"]), state=to64(s["state"]),
                scale=s["scale"] or s["q"].shape[-1] ** -0.5, lengths=None if s["lengths"] is None else s["lengths"].cpu())


def _check(s, grads=True):
    kw, k = _exact(s), _k(s)
    y, end = _call(s)
    (wy, wend), (my, mend) = oa.linear_attention(**kw), oa.linear_attention(mag=True, **kw)
    within(y, wy, my, k, "y")
    within(end, wend, mend, k, "state")
    if not grads:
        return
    names = [n for n in LEAVES if s[n] is not None]
    leaves = {n: s[n].detach().requires_grad_(True) for n in names}
    y2, end2 = _call(s, leaves)
    assert torch.equal(y2.detach(), y) and torch.equal(end2.detach(), end)
    got = dict(zip(names, torch.autograd.grad([y2, end2], list(leaves.values()), [s["dy"], s["dend"]])))
    dy, dend = to64(s["dy"]), to64(s["dend"])
    want, mag = oa.linear_attention_grad(dy, dend, **kw), oa.linear_attention_grad(dy, dend, mag=True, **kw)
    b, t, h = s["q"].shape[0], s["q"].shape[1], s["decay"].shape[-1]
    for n in names:
        assert got[n].dtype == s[n].dtype and got[n].shape == s[n].shape
        sums = b * t if n == "decay" and s["decay"].dim() == 1 else 2 * h + s["v"].shape[-1]
        within(got[n], want[n], mag[n], 2 * k + sums, "d" + n)


SHAPES = [(1, 1, 1, 1, 1), (2, 3, 2, 5, 7), (1, 16, 1, 16, 16), (1, 64, 2, 64, 64), (2, 65, 2, 64, 64), (1, 130, 3, 40, 72),
          (2, 33, 2, 128, 128), (1, 200, 2, 32, 16), (1, 257, 1, 100, 96), (3, 31, 4, 8, 8), (1, 300, 2, 64, 33),
          (2, 5, 2, 64, 64), (1, 90, 1, 128, 64), (1, 70, 2, 33, 128)]


@pytest.mark.parametrize("b,t,h,dk,dv", SHAPES)
@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_shapes_and_types(dev, b, t, h, dk, dv, dtype):
    _check(_make(dev, b, t, h, dk, dv, dtype=dtype))


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("dk,dv", [(32, 128), (7, 80), (64, 128), (48, 65), (128, 128)])
def test_more_than_64_values(dev, dtype, dk, dv):
    """Blocks of eight waves, in several segments, with shared heads and ends inside of them."""
    _check(_make(dev, 2, 330, 4, dk, dv, 2, 4, 2, dtype, ragged=True))


@pytest.mark.parametrize("h,hq,hk,hv", [(4, 4, 1, 1), (4, 2, 4, 2), (6, 1, 2, 3), (4, 1, 1, 4), (2, 2, 1, 2)])
@pytest.mark.parametrize("dtype,dk,dv", [(FP, 24, 40), (BF, 64, 128)])
@pytest.mark.parametrize("token", [True, False])
def test_shared_heads_and_decays(dev, h, hq, hk, hv, dtype, dk, dv, token):
    _check(_make(dev, 2, 70, h, dk, dv, hq, hk, hv, dtype, token))


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("b,h,t", [(65, 8, 130), (520, 1, 70)])
def test_sequences_in_one_piece(dev, dtype, b, h, t):
    """Enough heads that no sequence is cut into segments."""
    _check(_make(dev, b, t, h, 8, 8, dtype=dtype, token=False, ragged=True))


@pytest.mark.parametrize("t", [1, 30, 64, 150, 260])
@pytest.mark.parametrize("start", [True, False])
def test_ragged_batches(dev, t, start):
    s = _make(dev, 6, t, 2, 48, 32, hk=1, dtype=BF, start=start, ragged=True)
    s["lengths"][1], s["lengths"][2], s["lengths"][3] = 0, 1, t - 1
    _check(s)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_decays_of_all_sizes(dev, dtype):
    s = _make(dev, 2, 200, 4, 32, 32, dtype=dtype)
    # none, one in a million, one that forgets within a token, and a cleared state now and then
    s["decay"][..., 0], s["decay"][..., 1], s["decay"][..., 2] = 0.0, -1e-6, -40.0
    s["decay"][:, ::7, 3] = -float("inf")
    s["decay"][:, 3::29, 3] = -5000.0
    _check(s)
    y, end = _call(dict(s, decay=torch.full((4,), -float("inf"), device=dev)))
    alone = (s["q"].double() * s["k"].double()).sum(-1, keepdim=True) * s["v"].double() * 32 ** -0.5
    half = torch.finfo(dtype).eps / 2
    assert float((y.double() - alone).abs().max()) <= float(alone.abs().max()) * (half + 40 * 2.0 ** -18)
    # one product: of bf16 values exact in fp32; of fp32 ones six products of parts, added with a rounding each, without
    # the three below 2^-26 of it and what three parts leave of a factor, 2^-26 more: under eight half steps
    last = s["k"][:, -1, :, :, None].double() * s["v"][:, -1, :, None].double()
    assert float(((end.double() - last).abs() - (0 if dtype == BF else 8 * 2.0 ** -24) * last.abs()).max()) <= 0
    # a state that grows
    _check(dict(s, decay=torch.full((4,), 0.05, device=dev)))


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 128), (128, 48)])
def test_decay_gradients_keep_the_states_digits(dev, dtype, dk, dv):
    """States and their gradients that outweigh the tokens, all of one sign: a decay's gradient is then their product
    to within the roundings of fp32.  A lane adds 4 to 32 products, a wave 64 lanes' in 6 steps, then 4 waves' and up to
    2 tiles': 41; a chunk's step of either state rounds three times, over 7 chunks each: 42.  In 16 bits, where two parts
    of a state would be short of up to 2^-15 of it, that shows."""
    s = _make(dev, 2, 200, 2, dk, dv, dtype=dtype, rate=1e-3)
    for n in ("q", "k", "v", "dy"):
        s[n] = (s[n] * 2.0 ** -10).to(dtype)
    for n in ("state", "dend"):
        s[n] = 1 + s[n].abs()
    decay = s["decay"].detach().requires_grad_(True)
    _, end = _call(s, {"decay": decay})
    got, = torch.autograd.grad(end, decay, s["dend"])
    want = oa.linear_attention_grad(torch.zeros_like(to64(s["dy"])), to64(s["dend"]), **_exact(s))["decay"]
    assert float(((to64(got) - want) / want).abs().max()) <= 84 * 2.0 ** -24


def test_a_scale_of_ones_own(dev):
    _check(dict(_make(dev, 2, 70, 2, 32, 32, dtype=BF), scale=0.37))


def test_large_values_of_half_precision(dev):
    """Scores and states past fp16's range, outputs within it."""
    s = _make(dev, 1, 100, 2, 64, 64, dtype=HF, rate=0.01)
    s["q"], s["k"], s["v"] = (s["q"].float() * 400).to(HF), (s["k"].float() * 400).to(HF), (s["v"].float() * 1e-3).to(HF)
    s["dy"] = (s["dy"].float() * 1e-3).to(HF)
    s["state"] = s["state"] * 10
    kw = _exact(s)
    y, end = _call(s)
    (wy, wend), (my, mend) = oa.linear_attention(**kw), oa.linear_attention(mag=True, **kw)
    within(y, wy, my, _k(s), "y")
    within(end, wend, mend, _k(s), "state")


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_what_is_not_finite_does_not_reach_the_tokens_before(dev, dtype, bad):
    for key in ("v", "k", "q"):
        s = _make(dev, 1, 150, 2, 32, 48, dtype=dtype)
        clean, _ = _call(s)
        s[key][0, 90, 1, 5] = bad
        y, _ = _call(s)
        assert torch.equal(y[:, :, 0], clean[:, :, 0]) and torch.isfinite(y[0, :90]).all()
        kw, k = _exact(dict(s, **{key: torch.nan_to_num(s[key], 0, 0, 0)})), _k(s)
        wy, my = oa.linear_attention(**kw)[0], oa.linear_attention(mag=True, **kw)[0]
        within(y[:, :90], wy[:, :90], my[:, :90], k, key)
        if key == "v":                               # its column alone is lost
            cols = [i for i in range(48) if i != 5]
            assert torch.isfinite(y[0, :, 1][:, cols]).all() and not torch.isfinite(y[0, 90:, 1, 5]).any()


def test_what_stands_behind_a_sequence_is_not_read(dev):
    for t in (24, 200):
        s = _make(dev, 4, t, 2, 40, 40, dtype=BF, ragged=True)
        own = (t, 7, 0, t // 2 + 1)
        s["lengths"].copy_(torch.tensor(own))
        dirty = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        for i, n in enumerate(own):
            for k in ("q", "k", "v", "decay", "dy"):
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


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_strided_inputs(dev, dtype):
    s = _make(dev, 2, 70, 2, 32, 32, dtype=dtype)
    wide = torch.randn(2, 70, 400, device=dev).to(dtype)
    q, k, v = (wide[..., a:a + 64].unflatten(-1, (2, 32)) for a in (0, 64, 128))
    _check(dict(s, q=q, k=k, v=v))
    q, k, v = (wide[..., a:a + 64].unflatten(-1, (2, 32)) for a in (1, 67, 133))          # odd addresses
    _check(dict(s, q=q, k=k, v=v))
    # heads before tokens, every second value, one row for all sequences, a broadcast gradient
    t = {n: s[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k")}
    _check(dict(s, **t, v=wide[..., ::2][..., :64].unflatten(-1, (2, 32)), decay=s["decay"][:1].expand(2, 70, 2),
                dy=s["dy"][:1, :1].expand(2, 70, 2, 32)))
    _check(dict(s, decay=s["decay"].transpose(1, 2).contiguous().transpose(1, 2), q=s["q"][:, :, :1].expand(2, 70, 2, 32)))


def test_in_parts_equals_the_whole(dev):
    """A prompt in two parts and then token by token: the states that come back continue the sequence."""
    s = _make(dev, 3, 100, 4, 64, 48, hk=2, hv=2, dtype=BF)
    whole, end = _call(s)
    st, ys = s["state"], []
    for a, b in ((0, 16), (16, 85)):
        y, st = linear_attention(*(s[k][:, a:b] for k in ("q", "k", "v", "decay")), state=st, return_state=True)
        ys.append(y)
    for i in range(85, 100):
        nxt, before = torch.empty_like(st), st.clone()
        ys.append(linear_attention_step(st, *(s[k][:, i] for k in ("q", "k", "v", "decay")), out_state=nxt)[:, None])
        assert torch.equal(st, before)
        st = nxt
    my, mend = oa.linear_attention(mag=True, **_exact(s))
    k = 2 * _k(s)
    # both are within the bound of the exact values, y after a rounding to bf16 each
    within(st, to64(end), mend, k, "state")
    within(torch.cat(ys, 1), to64(whole), my + 1.02 * 2.0 ** 16 / k * to64(whole).abs(), k, "y")


@pytest.mark.parametrize("b,h,hq,hk,hv,dk,dv", [(1, 1, 1, 1, 1, 1, 1), (8, 16, 16, 4, 4, 64, 64), (5, 3, 1, 3, 1, 37, 6),
                                                (3, 4, 2, 1, 2, 128, 128), (2, 2, 2, 2, 2, 100, 70), (64, 2, 2, 2, 2, 32, 96),
                                                (2, 1, 1, 1, 1, 8, 65)])
@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("token", [True, False])
def test_step(dev, b, h, hq, hk, hv, dk, dv, dtype, token):
    s = _make(dev, b, 1, h, dk, dv, hq, hk, hv, dtype, token)
    kw = _exact(s)
    (wy, wend), (my, mend) = oa.linear_attention(**kw), oa.linear_attention(mag=True, **kw)
    cut = [s[k][:, 0] for k in ("q", "k", "v")] + [s["decay"][:, 0] if token else s["decay"]]
    st, out = s["state"].clone(), torch.full_like(s["state"], 9)
    y = linear_attention_step(st, *cut, out_state=out)
    assert torch.equal(st, s["state"])
    within(y, wy[:, 0], my[:, 0], 20 + dk, "y")
    within(out, wend, mend, 20, "state")
    y2 = linear_attention_step(st, *cut)
    assert torch.equal(y2, y) and torch.equal(st, out)                 # in place
    # views of a projection's rows, at odd addresses
    wide = torch.randn(b, (hq + hk) * dk + hk * dv + 3, device=dev).to(dtype)
    q = wide[:, 1:1 + hq * dk].unflatten(-1, (hq, dk))
    a, c = s["state"].clone(), s["state"].clone()
    y1 = linear_attention_step(a, q, *cut[1:])
    y2 = linear_attention_step(c, q.contiguous(), *cut[1:])
    assert torch.equal(y1, y2) and torch.equal(a, c)


def test_step_in_place_is_seen_by_a_graph_that_kept_the_state(dev):
    s = _make(dev, 2, 4, 2, 16, 16)
    k = s["k"].detach().requires_grad_(True)
    y = linear_attention(s["q"], k, s["v"], s["decay"], state=s["state"])
    linear_attention_step(s["state"], *(s[n][:, 0] for n in ("q", "k", "v", "decay")))
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


def test_empty_batches(dev):
    s = _make(dev, 2, 4, 2, 16, 8, dtype=BF)
    v = dict(s, **{k: s[k][:, :0] for k in ("q", "k", "v", "decay", "dy")})
    leaves = {k: v[k].detach().requires_grad_(True) for k in LEAVES}
    y, end = _call(v, leaves)
    assert y.shape == (2, 0, 2, 8) and torch.equal(end.detach(), s["state"])
    g = dict(zip(LEAVES, torch.autograd.grad([y, end], list(leaves.values()), [v["dy"], s["dend"]])))
    assert torch.equal(g["state"], s["dend"]) and g["q"].shape == (2, 0, 2, 16)
    y, end = _call(dict(s, **{k: s[k][:0] for k in ("q", "k", "v", "decay", "dy")}, state=None))
    assert y.shape == (0, 4, 2, 8) and end.shape == (0, 2, 16, 8)
    y = linear_attention_step(s["state"][:0], *(s[k][:0, 0] for k in ("q", "k", "v", "decay")))
    assert y.shape == (0, 2, 8)


def test_only_some_gradients(dev):
    s = _make(dev, 2, 90, 2, 32, 32, dtype=BF, start=False)
    full = {k: s[k].detach().requires_grad_(True) for k in LEAVES if s[k] is not None}
    ref = dict(zip(full, torch.autograd.grad(_call(s, full, want_state=False), list(full.values()), s["dy"])))
    for k in ("q", "v", "decay"):
        one = {k: s[k].detach().requires_grad_(True)}
        assert torch.equal(torch.autograd.grad(_call(s, one, want_state=False), one[k], s["dy"])[0], ref[k])
    leaf = s["k"].detach().requires_grad_(True)                       # the final state's gradient alone
    _, end = _call(s, {"k": leaf})
    got = torch.autograd.grad(end, leaf, s["dend"])[0]
    ckpt = ops.linear_attention(s["q"], s["k"], s["v"], s["decay"], want_checkpoints=True)[2]
    want = ops.linear_attention_grad(torch.zeros_like(s["dy"]), s["dend"], ckpt, s["q"], s["k"], s["v"], s["decay"], None,
                                     None, None)[1]
    assert torch.equal(got, want)


def test_equal_calls_give_equal_bits(dev):
    s = _make(dev, 2, 300, 4, 64, 64, hk=2, dtype=BF, token=False)
    runs = []
    for _ in range(3):
        leaves = {k: s[k].detach().requires_grad_(True) for k in LEAVES}
        y, end = _call(s, leaves)
        runs.append([y, end, *torch.autograd.grad([y, end], list(leaves.values()), [s["dy"], s["dend"]])])
    assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(runs[0], r))


def test_other_stream_and_graph(dev):
    s = _make(dev, 2, 150, 4, 64, 32, hk=2, dtype=BF, token=False)
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
            leaves["v"].copy_(torch.randn(2, 150, 4, 32, device=dev))
        ref = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref)), rep


def test_two_captured_calls_keep_apart(dev):
    """Prompts that need a workspace, captured in two graphs and replayed on two streams at once."""
    made = [_make(dev, 1, 900 + 100 * i, 4, 64, 64, dtype=BF, seed=i) for i in range(2)]
    want = [_call(s) for s in made]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s in made:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_call(s))
    streams = [torch.cuda.Stream(dev) for _ in made]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for o, w in zip(outs, want) for p, q in zip(o, w))


def test_saved_tensors_that_move(dev):
    """What a graph keeps may come back elsewhere and in another layout (offloaded activations)."""
    s = _make(dev, 2, 90, 4, 32, 32, hk=2, dtype=BF)
    wide = torch.randn(2, 90, 300, device=dev).to(BF)
    s.update(q=wide[..., 8:136].unflatten(-1, (4, 32)), k=wide[..., 137:201].unflatten(-1, (2, 32)))
    leaves = {k: s[k].detach().requires_grad_(True) for k in LEAVES}
    want = torch.autograd.grad(_call(s, leaves), list(leaves.values()), [s["dy"], s["dend"]])
    with torch.autograd.graph.save_on_cpu():
        out = _call(s, leaves)
    junk = [torch.full_like(wide, float("nan")) for _ in range(8)]
    got = torch.autograd.grad(out, list(leaves.values()), [s["dy"], s["dend"]])
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and len(junk) == 8


def test_refusals(dev):
    s = _make(dev, 2, 6, 4, 16, 8, hk=2, hv=2, dtype=BF)
    z = lambda *n, dt=BF: torch.zeros(*n, device=dev, dtype=dt)  # noqa: E731
    for err, kw in ((ValueError, dict(q=s["q"][0])), (ValueError, dict(k=s["k"][:, :5])), (TypeError, dict(k=s["k"].float())),
                    (ValueError, dict(k=s["k"][..., :8])), (ValueError, dict(v=z(2, 6, 3, 8))), (ValueError, dict(q=z(2, 6, 8, 16))),
                    (ValueError, dict(decay=s["decay"][:, :5])), (ValueError, dict(decay=s["decay"][0])),
                    (ValueError, dict(state=s["state"][..., :3])), (TypeError, dict(q=s["q"].to(HF))),
                    (ValueError, dict(q=z(2, 6, 4, 129), k=z(2, 6, 2, 129))), (ValueError, dict(v=z(2, 6, 2, 129))),
                    (ValueError, dict(v=z(2, 6, 2, 0))), (TypeError, dict(q=z(2, 6, 4, 16, dt=torch.float64),
                    k=z(2, 6, 2, 16, dt=torch.float64), v=z(2, 6, 2, 8, dt=torch.float64))), (RuntimeError, dict(v=s["v"].cpu()))):
        v = {**s, **kw}
        with pytest.raises(err):
            _call({**v, "state": v["state"] if "state" in kw else None})
    with pytest.raises(ValueError, match="lengths"):
        _call(dict(s, lengths=torch.ones(3, dtype=torch.int32, device=dev)))
    with pytest.raises(TypeError, match="lengths"):
        _call(dict(s, lengths=torch.ones(2, device=dev)))
    cut, st = [s[k][:, 0] for k in ("q", "k", "v", "decay")], s["state"]
    with pytest.raises(RuntimeError, match="no_grad"):
        linear_attention_step(st, cut[0].clone().requires_grad_(True), *cut[1:])
    with pytest.raises(ValueError, match="contiguous"):
        linear_attention_step(st.transpose(2, 3).contiguous().transpose(2, 3), *cut)
    with pytest.raises(TypeError, match="float32"):
        linear_attention_step(st.to(BF), *cut, out_state=torch.empty_like(st))
    with pytest.raises(ValueError):
        linear_attention_step(st, s["q"], *cut[1:])
    both = torch.zeros(3, 4, 16, 8, device=dev)
    with pytest.raises(ValueError, match="overlaps"):
        linear_attention_step(both[:2], *cut, out_state=both[1:])
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        dual = torch.autograd.forward_ad.make_dual(s["q"], torch.ones_like(s["q"]))
        linear_attention(dual, s["k"], s["v"], s["decay"])


def test_lengths_past_32_bits(dev):
    s = _make(dev, 3, 9, 2, 16, 16)
    outs = [_call(dict(s, lengths=v)) for v in (torch.tensor([2 ** 32 + 2, 4, -2 ** 33], device=dev),
                                                torch.tensor([9, 4, 0], dtype=torch.int32, device=dev))]
    assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_decays_and_states_in_other_types(dev):
    s = _make(dev, 2, 40, 2, 16, 16, dtype=BF)
    decay, state = s["decay"].to(BF).requires_grad_(True), s["state"].to(BF).requires_grad_(True)
    y, end = linear_attention(s["q"], s["k"], s["v"], decay, state=state, return_state=True)
    assert torch.equal(y.detach(), _call(dict(s, decay=decay.detach().float(), state=state.detach().float()))[0])
    g = torch.autograd.grad([y, end], [decay, state], [s["dy"], s["dend"]])
    assert g[0].dtype == BF and g[1].dtype == BF and end.dtype == FP


def test_a_cache_past_32_bit_offsets(dev):
    """Rows more than 2^32 elements into one buffer."""
    tokens, row = 70, 1 << 26
    big = torch.empty(tokens * row, dtype=BF, device=dev)
    views = [big.as_strided((1, tokens, 1, 32), (0, row, 32, 1), storage_offset=o) for o in (row - 96, row - 64, row - 32)]
    s = _make(dev, 1, tokens, 1, 32, 32, dtype=BF)
    for v, k in zip(views, ("q", "k", "v")):
        v.copy_(s[k])
    got = _call(dict(s, q=views[0], k=views[1], v=views[2]))
    assert all(torch.equal(p, q) for p, q in zip(got, _call(s)))
