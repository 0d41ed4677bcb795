"""Layer norm, short conv and selective scan where the other tests of single calls and modules do not go: prompts
of more than a hundred chunks, decay rates without a bound, NaN in the padding of a training batch, and the
gradients of padded products and of the conv behind a LayerNorm."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from ffnmem.memory.lngram_v2 import DepthwiseCausalConv
from ffnmem.memory.selective import SelectiveSSM
from oracle import memory as om
from oracle import mixing
from tests.bounds import within
from tests.test_gpu_selective import LEAVES, _call, _check, _make

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


# 32 tokens a chunk: 125 chunks, which all 16 waves of a joining block hold in one round, and 141 and 257 chunks,
# which take two and three rounds
@pytest.mark.parametrize("t", [4000, 4500, 8224])
def test_prompts_of_many_chunks(dev, t):
    _check(_make(dev, 2, t, 8, 4, dtype=FP, ragged=True))


@pytest.mark.parametrize("b,t,n", [(1, 17, 16), (2, 30, 20), (2, 30, 70), (3, 600, 5), (2, 600, 16), (1, 20, 40)])
def test_decay_rates_without_a_bound(dev, b, t, n):
    """A rate of minus infinity keeps nothing of the state before a token.  No time passes behind a sequence's end,
    where the product of the rate and a step of zero must not be formed."""
    s = _make(dev, b, t, 24, n, dtype=FP, ragged=b > 1)
    s["A"][::2, ::3] = float("-inf")
    s["A"][1::2, 1::3] = -3e38
    y, end = _call(s)
    v = {k: mixing.d(s[k]) for k in LEAVES}
    kw = dict(softplus=True, lengths=None if s["lengths"] is None else s["lengths"].cpu(), **v)
    (wy, wend), (my, mend) = mixing.selective_scan(**kw), mixing.selective_scan(mag=True, **kw)
    within(y, wy, my, 4 * t + 40, "y")
    within(end, wend, mend, 4 * t + 40, "state")
    names = [k for k in LEAVES if k not in ("dt", "dt_bias")]        # whose gradient is the rate times zero
    leaves = {k: s[k].detach().requires_grad_(True) for k in names}
    got = dict(zip(names, torch.autograd.grad(list(_call(s, leaves)), list(leaves.values()), [s["dy"], s["dend"]])))
    dy, dend = mixing.d(s["dy"]), mixing.d(s["dend"])
    want, mag = mixing.selective_grad(dy, dend, **kw), mixing.selective_grad(dy, dend, mag=True, **kw)
    sums = {"B": 24, "C": 24, "A": b * t, "D": b * t, "u": n, "z": n, "state": 0}
    for k in names:
        within(got[k], want[k], mag[k], 8 * t + 80 + sums[k], "d" + k)


# ----------------------------------------------------------------------------- the modules
def test_padding_of_a_training_batch_is_not_read(dev):
    """NaN embeddings behind the sequences' ends leave every gradient as it is."""
    torch.manual_seed(0)
    m = SelectiveSSM(32, 24).to(dev)
    emb = torch.randn(3, 20, 32, device=dev)
    own = torch.tensor([20, 6, 0], device=dev)
    dy = torch.randn(3, 20, 24, device=dev)
    runs = []
    for fill in (0.5, float("nan")):
        e = emb.clone()
        e[1, 6:], e[2] = fill, fill
        e.requires_grad_(True)
        y, (hist, scan) = m(e, lengths=own, return_state=True)
        g = torch.autograd.grad([y, hist, scan], [e, *m.parameters()], [dy, torch.ones_like(hist), torch.ones_like(scan)])
        runs.append([y, hist, scan, *g])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("d,n", [(72, 24), (100, 30), (96, 32)])
def test_products_of_odd_widths_and_their_gradients(dev, d, n):
    """The bf16 projections of ``SelectiveSSM``, padded where their rows are no multiple of 8 wide: sums of K, N and M
    products in fp32, one rounding each."""
    torch.manual_seed(1)
    m = SelectiveSSM(d, n).to(dev).to(BF)
    rows = 2 * 40
    for name, lin in (("w_in", m.w_in), ("w_x", m.w_x), ("w_dt", m.w_dt)):
        out, k = lin.weight.shape
        wide = torch.randn(2, 40, k + 3, device=dev).to(BF)
        x = wide[..., :k].detach().requires_grad_(True)        # rows longer than the product's, as a split leaves them
        dy = torch.randn(2, 40, out, device=dev).to(BF)
        y = m._linear(x, lin)
        dx, dw = torch.autograd.grad(y, [x, lin.weight], dy)
        x64, w64, d64 = (mixing.d(v) for v in (x, lin.weight, dy))
        within(y, x64 @ w64.t(), x64.abs() @ w64.t().abs(), k, name + " y")
        within(dx, d64 @ w64, d64.abs() @ w64.abs(), out, name + " dx")
        flat = d64.reshape(rows, out).t()
        within(dw, flat @ x64.reshape(rows, k), flat.abs() @ x64.reshape(rows, k).abs(), rows, name + " dw")
        with torch.no_grad():
            assert torch.equal(m._linear(x, lin), y)


@pytest.mark.parametrize("bias", [True, False])
def test_gradients_of_the_layer_norm_conv(dev, bias):
    """All three forms against autograd through the 64-bit restatement.  fp32: three sums of at most 60 roundings of
    2^-24 each one after the other, 1.1e-5 norm-relative."""
    torch.manual_seed(5)
    conv = DepthwiseCausalConv(48, 4, 3, 1e-5, normalization="LayerNorm", bias=bias, zero_init=False, device=dev)
    with torch.no_grad():
        for w in conv.norm.parameters():
            w.add_(torch.randn_like(w) * 0.2)
    x, dy = torch.randn(2, 25, 48, device=dev, requires_grad=True), torch.randn(2, 25, 48, device=dev)
    names = [k for k, _ in conv.named_parameters()]
    p = {k: mixing.d(v).requires_grad_(True) for k, v in conv.named_parameters()}
    x64 = mixing.d(x).requires_grad_(True)
    rows = F.layer_norm(x64, (48,), p["norm.weight"], p["norm.bias"], 1e-5)
    y64, _ = mixing.short_conv(rows, p["conv.weight"][:, 0], p.get("conv.bias"), 3, True)

    def parts(v):
        hist, ys = None, []
        for a, z in ((0, 4), (4, 5), (5, 25)):
            y, hist = conv.forward_incremental(v[:, a:z], hist)
            ys.append(y)
        return torch.cat(ys, 1)

    for got, want in ((conv(x), y64), (conv.forward_residual(x), x64 + y64), (parts(x), y64)):
        g = torch.autograd.grad(got, [x, *conv.parameters()], dy)
        ref = torch.autograd.grad(want, [x64, *(p[k] for k in names)], mixing.d(dy), retain_graph=True)
        for k, a, b in zip(["x", *names], g, ref):
            assert om.rel_err(a.cpu(), b) < 1.1e-5, k
