"""Autograd behaviour of the memory layer's norm and short conv modules, of the layer norm, the short conv and
the selective scan that they and ``SelectiveSSM`` run, on the CPU: the kernels are stood in for by the 64-bit
restatements, the autograd code around them is the library's own."""

from __future__ import annotations

import pytest
import torch

from ffnmem.memory.lngram_v2 import DepthwiseCausalConv
from lngram_hip import ops
from oracle import mixing


@pytest.fixture
def stand_ins(monkeypatch):
    """Kernels as functions of detached tensors, so that no graph passes through them that the library does not
    build itself."""

    def rmsnorm(x, w, eps, **_):
        x, w = x.detach(), w.detach()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w

    def short_conv(x, w, bias=None, dilation=1, silu=True, history=None, lengths=None, want_history=False):
        x, w, bias, history = (None if v is None else v.detach() for v in (x, w, bias, history))
        y, rows = mixing.short_conv(x, w, bias, dilation, silu, history, lengths)
        return (y, rows) if want_history else y

    monkeypatch.setattr(ops, "rmsnorm", rmsnorm)
    monkeypatch.setattr(ops, "short_conv", short_conv)


def test_rmsnorm_conv_with_a_bias_keeps_no_part_of_a_graph(stand_ins):
    """RMSNorm's kernel has no backward pass, so a graph behind it would lack the gradients of the rows and of
    the norm's weight without a word: the form is outside of autograd, as the one kernel of RMSNorm without a
    bias is."""
    torch.manual_seed(0)
    conv = DepthwiseCausalConv(6, 4, 2, 1e-5, bias=True, zero_init=False, dtype=torch.float64)
    x = torch.randn(2, 9, 6, dtype=torch.float64, requires_grad=True)
    past = torch.randn(2, 6, 6, dtype=torch.float64, requires_grad=True)
    whole = conv(x)
    assert not whole.requires_grad
    residual = conv.forward_residual(x)
    assert not residual.requires_grad and torch.equal(residual, x.detach() + whole)
    for history in (None, past):
        assert not any(t.requires_grad for t in conv.forward_incremental(x, history))
    with torch.no_grad():
        assert torch.equal(conv(x), whole) and torch.equal(conv.forward_residual(x), residual)
