"""The 64-bit forms of linear attention and group norm against autograd, differences and closed forms (CPU)."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as oa

F64 = torch.float64


def _make(b=2, t=7, h=4, hq=2, hk=2, hv=4, dk=3, dv=5, token=True, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=F64)

    decay = -torch.rand(*((b, t, h) if token else (h,)), generator=g, dtype=F64)
    return dict(q=r(b, t, hq, dk), k=r(b, t, hk, dk), v=r(b, t, hv, dv), g=decay, state=r(b, h, dk, dv)), r(b, t, h, dv), \
        r(b, h, dk, dv)


@pytest.mark.parametrize("token", [True, False])
@pytest.mark.parametrize("lengths", [None, torch.tensor([7, 3]), torch.tensor([0, 7])])
def test_gradients_are_those_of_the_forward_form(token, lengths):
    s, dy, dend = _make(token=token)
    leaves = {k: v.clone().requires_grad_(True) for k, v in s.items()}
    y, end = oa.linear_attention(leaves["q"], leaves["k"], leaves["v"], leaves["g"], 0.7, leaves["state"], lengths)
    want = torch.autograd.grad([y, end], list(leaves.values()), [dy, dend])
    got = oa.linear_attention_grad(dy, dend, s["q"], s["k"], s["v"], s["g"], 0.7, s["state"], lengths)
    for k, w in zip(("q", "k", "v", "decay", "state"), want):
        assert torch.allclose(got[k], w, rtol=1e-11, atol=1e-12), k
    mag = oa.linear_attention_grad(dy, dend, s["q"], s["k"], s["v"], s["g"], 0.7, s["state"], lengths, mag=True)
    assert all((mag[k] + 1e-12 >= got[k].abs()).all() for k in got)


def test_a_decay_by_differences():
    s, dy, dend = _make(token=True)
    got = oa.linear_attention_grad(dy, dend, s["q"], s["k"], s["v"], s["g"], 0.7, s["state"])["decay"]

    def loss(g):
        y, end = oa.linear_attention(s["q"], s["k"], s["v"], g, 0.7, s["state"])
        return (y * dy).sum() + (end * dend).sum()

    for at in ((0, 0, 1), (1, 3, 0), (0, 6, 3)):
        up, down = s["g"].clone(), s["g"].clone()
        up[at] += 1e-5
        down[at] -= 1e-5
        assert abs(float((loss(up) - loss(down)) / 2e-5 - got[at])) < 1e-7


def test_closed_forms():
    """No decay: a running sum of outer products; a cleared state: each token alone."""
    s, _, _ = _make(h=4, hq=4, hk=4, hv=4)
    y, end = oa.linear_attention(s["q"], s["k"], s["v"], torch.zeros(4, dtype=F64), 1.0)
    w = torch.einsum("bihk,bjhk->bhij", s["q"], s["k"]).tril()
    assert torch.allclose(y, torch.einsum("bhij,bjhv->bihv", w, s["v"]))
    assert torch.allclose(end, torch.einsum("bthk,bthv->bhkv", s["k"], s["v"]))
    y, _ = oa.linear_attention(s["q"], s["k"], s["v"], torch.full((4,), -float("inf"), dtype=F64), 1.0, s["state"])
    assert torch.allclose(y, (s["q"] * s["k"]).sum(-1, keepdim=True) * s["v"])


@pytest.mark.parametrize("shape,groups", [((4, 12), 3), ((3, 5, 12), 3), ((2, 4, 3, 8), 8), ((2, 6, 8), 1)])
@pytest.mark.parametrize("silu", [True, False])
def test_group_norm_is_torchs(shape, groups, silu):
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(s, generator=g, dtype=F64) for s in (shape, shape[-1:], shape[-1:], shape))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    moved = leaves[0].movedim(-1, 1)
    z = torch.nn.functional.group_norm(moved, groups, leaves[1], leaves[2], 1e-5).movedim(1, -1)
    y = torch.nn.functional.silu(z) if silu else z
    want = torch.autograd.grad(y, leaves, dy)
    assert torch.allclose(oa.group_norm(x, groups, w, b, 1e-5, silu), y)
    for p, q, m in zip(oa.group_norm_grad(dy, x, groups, w, b, 1e-5, silu), want,
                       oa.group_norm_grad(dy, x, groups, w, b, 1e-5, silu, mag=True)):
        assert torch.allclose(p, q, rtol=1e-10, atol=1e-12) and (m + 1e-12 >= p.abs()).all()
    assert (oa.group_norm(x, groups, w, b, 1e-5, silu, mag=True) + 1e-12 >= y.detach().abs()).all()
