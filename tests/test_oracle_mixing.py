"""The 64-bit forms of layer norm, the short conv and the selective scan (``oracle/mixing.py``): their
gradient formulas against autograd and against differences (CPU)."""

from __future__ import annotations

import pytest
import torch

from oracle import mixing

F64 = torch.float64


def _r(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, dtype=F64) * std


def test_layer_norm_grad():
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = _r(g, 5, 7).requires_grad_(True), _r(g, 7).requires_grad_(True), _r(g, 7).requires_grad_(True), _r(g, 5, 7)
    y = mixing.layer_norm(x, w, b, 1e-5)
    assert torch.allclose(y, torch.nn.functional.layer_norm(x, (7,), w, b, 1e-5), atol=1e-13)
    want = torch.autograd.grad(y, (x, w, b), dy)
    for got, ref in zip(mixing.layer_norm_grad(dy, x.detach(), w.detach(), 1e-5), want):
        assert torch.allclose(got, ref, atol=1e-12)


def test_short_conv_is_the_convolution():
    g = torch.Generator().manual_seed(2)
    x, w, b = _r(g, 2, 11, 3), _r(g, 3, 4), _r(g, 3)
    y, hist = mixing.short_conv(x, w, b, 2, False)
    ref = torch.nn.functional.conv1d(torch.nn.functional.pad(x.transpose(1, 2), (6, 0)), w[:, None], b, dilation=2,
                                     groups=3).transpose(1, 2)
    assert torch.allclose(y, ref, atol=1e-13)
    # in two parts, the second from the first one's history
    y1, h1 = mixing.short_conv(x[:, :4], w, b, 2, True)
    y2, h2 = mixing.short_conv(x[:, 4:], w, b, 2, True, h1)
    assert torch.allclose(torch.cat((y1, y2), 1), mixing.short_conv(x, w, b, 2, True)[0]) and torch.equal(h2, hist)


@pytest.mark.parametrize("softplus,gated", [(True, True), (False, False)])
def test_selective_grad(softplus, gated):
    g = torch.Generator().manual_seed(3)
    b, t, c, n, gr = 3, 6, 4, 3, 2
    ins = dict(u=_r(g, b, t, c), dt=_r(g, b, t, c, std=0.3), A=-_r(g, c, n).abs(), B=_r(g, b, t, gr, n),
               C=_r(g, b, t, gr, n), D=_r(g, c), z=_r(g, b, t, c), dt_bias=_r(g, c), state=_r(g, b, c, n))
    if not gated:
        ins["z"] = None
    lengths = torch.tensor([6, 4, 0])
    dy, dend = _r(g, b, t, c), _r(g, b, c, n)

    def loss(**kw):
        y, end = mixing.selective_scan(softplus=softplus, lengths=lengths, **kw)
        return (y * dy).sum() + (end * dend).sum()

    leaves = {k: v.clone().requires_grad_(True) for k, v in ins.items() if v is not None}
    want = dict(zip(leaves, torch.autograd.grad(loss(**{**ins, **leaves}), list(leaves.values()), allow_unused=True)))
    got = mixing.selective_grad(dy, dend, softplus=softplus, lengths=lengths, **ins)
    for k in leaves:
        assert torch.allclose(got[k], want[k], atol=1e-12), k
    # and against differences
    with torch.no_grad():
        for k in leaves:
            v, h = _r(g, *ins[k].shape), 1e-6
            diff = (loss(**{**ins, k: ins[k] + h * v}) - loss(**{**ins, k: ins[k] - h * v})) / (2 * h)
            assert abs(float(diff - (got[k] * v).sum())) < 1e-6 * (1 + abs(float(diff))), k
        mags = mixing.selective_grad(dy, dend, softplus=softplus, lengths=lengths, mag=True, **ins)
        assert all((mags[k] >= got[k].abs() - 1e-12).all() for k in leaves)
