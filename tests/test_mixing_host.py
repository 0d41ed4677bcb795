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


def _dual(*shape):
    return torch.autograd.forward_ad.make_dual(torch.randn(*shape), torch.randn(*shape))


def test_forward_mode_tangents_are_refused():
    """The operators have no forward-mode derivative.  A tangent asks for no reverse-mode graph, so it would be
    dropped on the way to the kernel, under no_grad too."""
    from ffnmem.memory.norm import LayerNorm, layer_norm
    from ffnmem.memory.selective import SelectiveSSM, selective_scan, selective_step
    from ffnmem.memory.short_conv import short_conv, short_conv_step

    def r(*s):
        return torch.randn(*s)

    scan = dict(u=(1, 3, 4), dt=(1, 3, 4), A=(4, 2), B=(1, 3, 2), C=(1, 3, 2), D=(4,), z=(1, 3, 4), dt_bias=(4,),
                state=(1, 4, 2))
    step = dict(state=(1, 4, 2), u=(1, 4), dt=(1, 4), A=(4, 2), B=(1, 2), C=(1, 2), D=(4,), z=(1, 4), dt_bias=(4,))
    conv = dict(x=(1, 3, 4), weight=(4, 2), bias=(4,), history=(1, 1, 4))
    one = dict(x=(1, 4), history=(1, 1, 4), weight=(4, 2), bias=(4,))
    norm = dict(x=(3, 4), weight=(4,), bias=(4,))
    with torch.autograd.forward_ad.dual_level():
        for fn, shapes in ((layer_norm, norm), (short_conv, conv), (short_conv_step, one), (selective_scan, scan),
                           (selective_step, step)):
            for name in shapes:
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                        fn(**{k: _dual(*s) if k == name else r(*s) for k, s in shapes.items()})
        for fn in (LayerNorm(4), DepthwiseCausalConv(4, 2, 1, 1e-5, normalization="LayerNorm"), SelectiveSSM(4, 4)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(_dual(1, 3, 4))
        with pytest.raises(RuntimeError, match="no CPU path"):   # inside a level, without a tangent: as ever
            layer_norm(r(3, 4), r(4))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(layer_norm, (r(3, 4),), (r(3, 4),))


def test_one_kernel_forms_of_the_conv():
    """Which norm and bias a conv has is read as they are now: replaced and parametrised ones too."""
    conv = DepthwiseCausalConv(4, 2, 1, 1e-5)
    assert conv.one_kernel
    torch.nn.utils.parametrizations.weight_norm(conv.conv)
    assert conv.one_kernel
    conv.conv.bias = torch.nn.Parameter(torch.zeros(4))
    assert not conv.one_kernel
    torch.nn.utils.parametrize.register_parametrization(conv.conv, "bias", torch.nn.Identity())
    assert "bias" not in conv.conv._parameters and not conv.one_kernel
    conv = DepthwiseCausalConv(4, 2, 1, 1e-5)
    conv.norm = DepthwiseCausalConv(4, 2, 1, 1e-5, normalization="LayerNorm").norm
    assert not conv.one_kernel
