"""Layer norm and its backward pass (``lng_layer_norm``, ``lng_layer_norm_grad``) against the 64-bit form."""

from __future__ import annotations

import pytest
import torch

from tests.bounds import U32, within
from ffnmem.memory.lngram_v2 import build_lngram_norm
from ffnmem.memory.norm import LayerNorm, layer_norm
from lngram_hip import ops
from oracle import mixing

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (130, 32), (33, 40), (7, 128), (65, 256), (9, 512), (1000, 1024), (5, 2048),
          (3, 2056), (6, 4096), (2, 8192), (2, 8200), (3, 1000), (17, 37), (300, 64), (2049, 96)]


def _k(rows: int, d: int) -> float:
    """Roundings of one sum: a thread adds at most 32 elements (d / 256 of them past 8192 and for rows that
    are not 16-byte pieces), a dozen more join the threads; then some ten steps of the formula.  Statistics
    (mean, variance) and a sum over them: three such sums on a result's way."""
    return 3 * (max(32, d / 256) + 12) + 10


def _k_cols(rows: int) -> float:
    """A column's sum adds at most every row one after the other."""
    return rows + 160


def _make(dev, rows, d, dtype, wt, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, d, generator=g) + mean * torch.randn(rows, 1, generator=g)).to(dtype).to(dev)
    w = b = None
    if wt is not None:
        w, b = (1 + 0.3 * torch.randn(d, generator=g)).to(wt).to(dev), torch.randn(d, generator=g).to(wt).to(dev)
    return x, w, b, torch.randn(rows, d, generator=g).to(dtype).to(dev)


def _check(x, w, b, dy, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    have = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(y, have, dy)))
    assert torch.equal(y.detach(), layer_norm(x, w, b, eps))          # with and without a graph
    xd, wd, bd, gd = (mixing.d(t) for t in (x, w, b, dy))
    rows, d = x.numel() // x.shape[-1], x.shape[-1]
    within(y, mixing.layer_norm(xd, wd, bd, eps), mixing.layer_norm_mag(xd, wd, bd, eps) + 0 * xd, _k(rows, d), "y")
    want, mag = mixing.layer_norm_grad(gd, xd, wd, eps), mixing.layer_norm_grad_mag(gd, xd, wd, eps)
    for i, name, k in ((0, "dx", _k(rows, d)), (1, "dw", _k_cols(rows)), (2, "db", _k_cols(rows))):
        if i in grads:
            assert grads[i].dtype == leaves[i].dtype
            within(grads[i], want[i], mag[i], k, name)


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("dtype,wt", [(BF, BF), (BF, FP), (FP, FP), (HF, HF), (HF, FP), (FP, None)])
def test_shapes_and_types(dev, rows, d, dtype, wt):
    _check(*_make(dev, rows, d, dtype, wt, seed=rows + d))


@pytest.mark.parametrize("d", [1, 2, 15, 17, 63, 65, 255, 257, 511, 513, 1023, 1025, 2047, 2050, 4095, 4097, 8191])
@pytest.mark.parametrize("rows,dtype,wt", [(37, BF, FP), (70, FP, FP), (1, HF, HF)])
def test_odd_widths(dev, d, rows, dtype, wt):
    """Each side of the widths at which a row is held by more threads, one element a load."""
    _check(*_make(dev, rows, d, dtype, wt, seed=rows + d))


def test_weight_or_bias_alone(dev):
    x, w, b, dy = _make(dev, 40, 256, BF, FP)
    _check(x, w, None, dy)
    _check(x, None, b, dy)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strided_and_misaligned_rows(dev, dtype):
    x, w, b, dy = _make(dev, 60, 128, dtype, dtype)
    wide = torch.randn(60, 200, device=dev).to(dtype)
    _check(wide[:, 8:136], w, b, dy)                                  # a part of wider rows
    _check(wide[:, 3:131], w, b, dy)                                  # one whose address is not a 16-byte multiple
    _check(wide[::2, 8:136], w, b, dy[:30])
    _check(x.view(3, 20, 128).transpose(0, 1), w, b, dy.view(3, 20, 128).transpose(0, 1))   # rows that do not collapse
    _check(x[:1].expand(60, 128), w, b, dy)                           # the same row again and again
    _check(x, w, b, dy[:1].expand(60, 128))
    _check(wide[:, :120].t().contiguous().t(), *_make(dev, 60, 120, dtype, dtype)[1:])      # columns contiguous
    big_w = torch.randn(300, device=dev).to(dtype)
    _check(x, big_w[1:129], big_w[5:133], dy)                         # weights at odd addresses


def test_large_means_and_constant_rows(dev):
    x, w, b, dy = _make(dev, 50, 1024, FP, FP, mean=300.0)
    _check(x, w, b, dy)
    c = torch.full((4, 512), 3.0, device=dev)
    y = layer_norm(c, None, None, 1e-5)
    assert torch.equal(y, torch.zeros_like(y))                        # (x - mean) is exactly zero
    z = torch.zeros(4, 512, device=dev, dtype=BF)
    assert torch.equal(layer_norm(z, None, None, 0.0).isnan(), torch.ones_like(z, dtype=torch.bool))  # 0 / 0, as defined


def test_a_bad_row_stays_alone(dev):
    x, w, b, dy = _make(dev, 64, 256, BF, BF)
    ok = layer_norm(x, w, b)
    bad = x.clone()
    bad[7, 3], bad[20, 0] = float("nan"), float("inf")
    y = layer_norm(bad, w, b)
    keep = torch.ones(64, dtype=torch.bool, device=dev)
    keep[7] = keep[20] = False
    assert torch.equal(y[keep], ok[keep]) and y[~keep].isnan().all()


def test_no_rows_and_many_rows(dev):
    x, w, b, _ = _make(dev, 1, 64, BF, FP)
    e = x[:0].requires_grad_(True)
    wl, bl = w.requires_grad_(True), b.requires_grad_(True)
    y = layer_norm(e, wl, bl)
    dx, dw, db = torch.autograd.grad(y, (e, wl, bl), torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64)
    assert torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, torch.zeros_like(db))
    # more rows than a launch's blocks take in one round, and offsets past 2^31 bytes
    n, d = 600_001, 2048
    x = torch.randn(1024, d, device=dev).to(BF)
    xl = x.repeat(n // 1024 + 1, 1)[:n]
    y = layer_norm(xl)
    assert torch.equal(y[-(n % 1024):], layer_norm(x)[:n % 1024])
    assert torch.equal(y[512 * 1024:513 * 1024], layer_norm(x))
    del xl, y


def test_equal_calls_give_equal_bits(dev):
    x, w, b, dy = _make(dev, 3001, 1024, BF, FP)
    y, mean, rstd = ops.layer_norm(x, w, b, 1e-5, want_stats=True)
    first = ops.layer_norm_grad(dy, x, w, mean, rstd)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, ops.layer_norm_grad(dy, x, w, mean, rstd)))


def test_gradient_against_differences(dev):
    x, w, b, dy = _make(dev, 12, 96, FP, FP)
    _, mean, rstd = ops.layer_norm(x, w, b, 1e-5, want_stats=True)
    grads = ops.layer_norm_grad(dy, x, w, mean, rstd)
    xd, wd, bd, gd = (mixing.d(t) for t in (x, w, b, dy))
    g, h = torch.Generator().manual_seed(5), 1e-6
    for i, (grad, at) in enumerate(zip(grads, (xd, wd, bd))):
        v = torch.randn(at.shape, generator=g, dtype=torch.float64)
        f = [(mixing.layer_norm(*[t + s * h * v if j == i else t for j, t in enumerate((xd, wd, bd))], 1e-5) * gd).sum()
             for s in (1, -1)]
        mag = mixing.layer_norm_grad_mag(gd, xd, wd, 1e-5)[i]
        # the difference quotient's own error: h^2 and 2^-53 / h
        assert abs(float((f[0] - f[1]) / (2 * h) - (mixing.d(grad) * v).sum())) < \
            _k_cols(12 * 96) * U32 * float((mag * v.abs()).sum()) + 1e-6


def test_other_stream_and_graph(dev):
    x, w, b, dy = _make(dev, 512, 128, FP, FP)
    want = [layer_norm(x, w, b)]
    st = torch.cuda.Stream(dev)
    st.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(st):
        got = layer_norm(x, w, b)
    torch.cuda.current_stream(dev).wait_stream(st)
    assert torch.equal(got, want[0])
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(512, 128, device=dev))
        ref = step()                                                  # eager work between the replays
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref)), rep


def test_module(dev):
    m = build_lngram_norm("LayerNorm", 96, 1e-5, dev, BF)
    assert isinstance(m, LayerNorm) and set(m.state_dict()) == {"weight", "bias"}
    x = torch.randn(2, 5, 96, device=dev).to(BF)
    assert torch.equal(m(x), layer_norm(x, m.weight.detach(), m.bias.detach(), 1e-5))
    with pytest.raises(ValueError, match="last dim 96"):
        m(x[..., :95])


def test_refusals(dev):
    x, w, b, dy = _make(dev, 4, 64, BF, BF)
    for args, err in (((x.double(), w, b, 1e-5), TypeError), ((x, w.to(HF), b.to(HF), 1e-5), TypeError),
                      ((x, w.float(), b, 1e-5), TypeError), ((x.float(), w, b, 1e-5), TypeError),
                      ((x, w[:63], b, 1e-5), ValueError), ((x, w, b[None], 1e-5), ValueError),
                      ((x[:, :0], None, None, 1e-5), ValueError), ((x, w.cpu(), b, 1e-5), RuntimeError)):
        with pytest.raises(err):
            layer_norm(*args)
    _, mean, rstd = ops.layer_norm(x, w, b, 1e-5, want_stats=True)
    with pytest.raises(ValueError):
        ops.layer_norm_grad(dy[:3], x, w, mean, rstd)
    with pytest.raises(TypeError):
        ops.layer_norm_grad(dy.float(), x, w, mean, rstd)
    with pytest.raises(ValueError):
        ops.layer_norm_grad(dy, x, w, mean[:3], rstd)
    y = layer_norm(x.requires_grad_(True), w, b)
    (gx,) = torch.autograd.grad((y.float() ** 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.float().sum().backward()
