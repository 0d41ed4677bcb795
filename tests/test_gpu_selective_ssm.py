"""``SelectiveSSM`` as the token router's SSM context (whole sequences, training, decoding), and the memory
layer with LayerNorm and a conv bias, against 64-bit restatements.

fp32 outputs are within 1e-5 (norm-relative) of 64 bits and bf16 ones within 2e-2, as the memory layer's own
are; fp32 gradients pass six sums of at most 300 roundings of 2^-24 each: 1.1e-4."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from ffnmem import infer
from ffnmem.memory.lngram_v2 import DepthwiseCausalConv, RMSNorm
from ffnmem.memory.norm import LayerNorm
from ffnmem.memory.selective import SelectiveSSM
from ffnmem.memory.wrapper import LngramMemory
from oracle import memory as om
from oracle import mixing

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


# ----------------------------------------------------------------------------- SelectiveSSM
def _ssm(dev, d=128, n=48, dtype=FP, seed=0):
    torch.manual_seed(seed)
    m = SelectiveSSM(d, n, d_state=16)
    with torch.no_grad():                            # weights of a trained size: every term of the output counts
        m.w_in.weight.normal_(0, d ** -0.5)
        m.w_x.weight.normal_(0, n ** -0.5)
        m.norm.weight.normal_(1, 0.2)
        m.norm.bias.normal_(0, 0.2)
    return m.to(dtype).to(dev)


def _restated(p: dict, m: SelectiveSSM, emb, lengths=None, state=None):
    x = F.layer_norm(emb, emb.shape[-1:], p["norm.weight"], p["norm.bias"], m.norm.eps)
    x, z = F.linear(x, p["w_in.weight"]).chunk(2, -1)
    hist, scan = (None, None) if state is None else state
    u, hist = mixing.short_conv(x, p["conv.weight"][:, 0], p["conv.bias"], 1, True, hist, lengths)
    low, bm, cm = F.linear(u, p["w_x.weight"]).split((m.dt_rank, m.d_state, m.d_state), -1)
    y, scan = mixing.selective_scan(u, F.linear(low, p["w_dt.weight"]), -torch.exp(p["A_log"]), bm[:, :, None],
                                    cm[:, :, None], p["D"], z, p["dt_bias"], True, scan, lengths)
    return y, (hist, scan)


def _params(m) -> dict:
    return {k: mixing.d(v) for k, v in m.named_parameters()}


def test_forward_and_gradients(dev):
    m = _ssm(dev)
    g = torch.Generator().manual_seed(3)
    emb = torch.randn(3, 50, 128, generator=g)
    lengths = torch.tensor([50, 20, 0], dtype=torch.int32)
    dy = torch.randn(3, 50, 48, generator=g)
    e = emb.to(dev).requires_grad_(True)
    y, (hist, scan) = m(e, lengths=lengths.to(dev), return_state=True)
    with torch.no_grad():
        assert torch.equal(m(e, lengths=lengths.to(dev)), y)
    p = {k: v.requires_grad_(True) for k, v in _params(m).items()}
    e64 = emb.double().requires_grad_(True)
    want, (whist, wscan) = _restated(p, m, e64, lengths)
    assert om.rel_err(y.detach().cpu(), want.detach()) < 1e-5
    assert om.rel_err(hist.detach().cpu(), whist.detach()) < 1e-5 and om.rel_err(scan.detach().cpu(), wscan.detach()) < 1e-5
    assert (y[2] == 0).all() and (y[1, 20:] == 0).all()
    names = list(p)
    got = torch.autograd.grad(y, [e, *(dict(m.named_parameters())[k] for k in names)], dy.to(dev))
    ref = torch.autograd.grad(want, [e64, *(p[k] for k in names)], dy.double())
    for k, a, b in zip(["emb", *names], got, ref):
        assert om.rel_err(a.cpu(), b) < 1.1e-4, k


@pytest.mark.parametrize("dtype,tol", [(FP, 1e-5), (BF, 2e-2)])
def test_parts_and_steps_continue_a_sequence(dev, dtype, tol):
    m = _ssm(dev, dtype=dtype)
    emb = torch.randn(2, 40, 128, generator=torch.Generator().manual_seed(4)).to(dtype).to(dev)
    with torch.no_grad():
        whole, end = m(emb, return_state=True)
        y, st = m(emb[:, :17], return_state=True)
        ys = [y]
        kept = [t.clone() for t in st]
        y2, st2 = m(emb[:, 17:30], state=st, return_state=True)
        assert all(torch.equal(a, b) for a, b in zip(st, kept))     # the given state stays: a way back
        ys.append(y2)
        for i in range(30, 40):
            y, st2 = m.step(st2, emb[:, i])
            ys.append(y[:, None])
        one, _ = m.step(None, emb[:, 0])
    assert om.rel_err(torch.cat(ys, 1).float().cpu(), whole.float().cpu()) < tol
    assert om.rel_err(one.float().cpu(), whole[:, 0].float().cpu()) < tol
    assert om.rel_err(st2[1].cpu(), end[1].cpu()) < tol
    want, _ = _restated(_params(m), m, mixing.d(emb))
    assert om.rel_err(whole.float().cpu(), want) < tol


@pytest.mark.parametrize("d,n", [(72, 24), (100, 30)])
def test_bf16_training_of_odd_widths(dev, d, n):
    """Widths and ranks that are no multiple of 8: features as fp32 weights of the same values give them, and
    gradients of all parameters, from ragged sequences' features and both parts of the state."""
    m = _ssm(dev, d, n, BF)
    emb = torch.randn(2, 40, d, device=dev).to(BF)
    own = torch.tensor([40, 7], device=dev)
    y, (hist, scan) = m(emb, lengths=own, return_state=True)
    assert y.dtype == BF and scan.dtype == FP and bool((y[1, 7:] == 0).all())
    wide = SelectiveSSM(d, n).to(dev)
    wide.load_state_dict(m.state_dict())
    assert om.rel_err(y.detach().float().cpu(), wide(emb.float(), lengths=own).detach().cpu()) < 2e-2
    (y.float().sum() + hist.float().sum() + scan.sum()).backward()
    for k, p in m.named_parameters():
        assert p.grad.shape == p.shape and p.grad.dtype == BF and bool(torch.isfinite(p.grad).all()), k


def test_no_tokens_and_no_sequences(dev):
    m = _ssm(dev)
    emb = torch.randn(2, 5, 128, device=dev)
    with torch.no_grad():
        _, state = m(emb, return_state=True)
        y, after = m(emb[:, :0], state=state, return_state=True)
        assert y.shape == (2, 0, 48) and all(torch.equal(p, q) for p, q in zip(after, state))
        assert m(emb[:0]).shape == (0, 5, 48)
    y, after = m(emb[:, :0], state=state, return_state=True)
    grads = torch.autograd.grad(y.sum() + after[1].sum(), list(m.parameters()), allow_unused=True)
    assert all(g is None or bool((g == 0).all()) for g in grads)


def test_step_replayed_from_a_graph(dev):
    m = _ssm(dev, dtype=BF)
    emb = torch.randn(4, 128, device=dev).to(BF)
    state = tuple(t.clone() for t in m.empty_state(4))

    def step():
        with torch.no_grad():
            y, new = m.step(state, emb)
            for a, b in zip(state, new):
                a.copy_(b)
        return y

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    ref_state = None
    for a, b in zip(state, m.empty_state(4)):
        a.copy_(b)
    for rep in range(4):
        emb.copy_(torch.randn(4, 128, device=dev))
        ref, ref_state = m.step(ref_state, emb)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and all(torch.equal(a, b) for a, b in zip(state, ref_state)), rep


def test_context_of_the_token_router(dev):
    """The memory layer routed by the selective features: a whole sequence at once, and decoded token by token
    with the features, the code cache and the conv cache moving on together."""
    torch.manual_seed(1)
    d, v, b, t = 128, 200, 2, 20
    cfg = {"routes": 8, "mem_dim": 32, "kv_heads": 2, "q_heads": 4, "head_dim": 32, "router_input": "embed2_ssm",
           "execution_mode": "full"}
    mem = LngramMemory(d, cfg, ssm_dim=48)
    with torch.no_grad():
        mem.module.readout_o_proj.weight.normal_(0, 0.02)
        mem.module.short_conv.conv.weight.normal_(0, 0.2)
    mem = mem.to(dev).eval()
    ssm = _ssm(dev)
    table = torch.randn(v, d, device=dev) * 0.02
    tok = torch.randint(0, v, (b, t), device=dev)
    h = torch.randn(b, t, d, device=dev)
    model = infer.memory_model(mem, tok_emb=lambda ids: table[ids], ssm=ssm)
    with torch.no_grad():
        feats = ssm(table[tok])
        whole = mem.forward_ids(h, tok, table, feats)
        codes = mem.route_codes(mem.router_features(table[tok], feats))[1]
        st = infer.DecodeState.empty(model, b, t)
        sst, outs = None, []
        for i in range(t):
            f, sst = ssm.step(sst, table[tok[:, i]])
            assert om.rel_err(f.cpu(), feats[:, i].cpu()) < 1e-5
            x = infer.router_input_at(model, mem, st, table[tok[:, i:i + 1]], f[:, None])
            assert x.shape == (b, 1, 2 * d + 48)
            # the codes of the whole sequence: a logit next to zero may change its sign with the last bit
            outs.append(infer.memory_step(model, 0, st, h[:, i:i + 1].contiguous(), codes[:, i:i + 1]))
            st.tokens[:, i] = tok[:, i]
            st.ssm[:, i] = f
            st.length += 1
        assert om.rel_err(torch.cat(outs, 1).cpu(), whole.cpu()) < 1e-5
    for fn in (lambda: infer.ssm_continue(model, h, None), lambda: infer.tree_ssm_states(model, st, h[:, :2], [-1, 0])):
        with pytest.raises(NotImplementedError, match="SelectiveSSM"):
            fn()


# ----------------------------------------------------------------------------- the layer with LayerNorm / bias
def _layer(dev, dtype, norm, bias, d=128, seed=2):
    torch.manual_seed(seed)
    sb = d == 1024
    cfg = {"routes": 184 if sb else 8, "mem_dim": 128 if sb else 32, "kv_heads": 4 if sb else 2,
           "q_heads": 16 if sb else 4, "head_dim": 64 if sb else 32, "normalization": norm, "conv_bias": bias,
           "execution_mode": "full"}
    mem = LngramMemory(d, cfg)
    m = mem.module
    with torch.no_grad():
        m.readout_o_proj.weight.normal_(0, 0.02)
        m.short_conv.conv.weight.normal_(0, 0.2)
        for n, w in m.named_parameters():
            if "norm" in n or n.endswith("conv.bias"):
                w.add_(torch.randn_like(w) * 0.2)
    return mem.to(dtype).to(dev).eval()


def _norm64(p, key, x, eps):
    if key + ".bias" in p:
        return F.layer_norm(x, x.shape[-1:], p[key + ".weight"], p[key + ".bias"], eps)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * p[key + ".weight"]


def _layer64(mem, h, codes):
    m = mem.module
    p = {k: mixing.d(v) for k, v in m.state_dict().items()}
    cfg = om.MemCfg(m.hidden_size, m.num_routes, m.memory_dim, m.readout_num_heads, m.readout_num_kv_heads,
                    m.readout_head_dim, eps=m.readout_query_norm.eps)
    h, codes = mixing.d(h), codes.cpu().numpy().astype("int32")
    b, t, _ = h.shape
    q = F.linear(_norm64(p, "readout_query_norm", h, cfg.eps), p["readout_q_proj.weight"])
    tok = om.route_tokens({n: p[f"tables.ngram_{n}.weight"] for n in cfg.orders}, codes, cfg.orders, cfg.bits)
    kv = F.linear(_norm64(p, "readout_memory_norm", tok, cfg.eps), p["readout_kv_proj.weight"])
    shape = (b, t, m.num_routes, cfg.kv_heads, cfg.head_dim)
    key, value = (x.reshape(shape).permute(0, 1, 3, 2, 4) for x in kv.chunk(2, -1))
    head = om.manual_gqa(cfg, q.view(b, t, cfg.q_heads, cfg.head_dim), key, value)
    mixed = F.linear(head.reshape(b, t, -1), p["readout_o_proj.weight"])
    conv, _ = mixing.short_conv(_norm64(p, "short_conv.norm", mixed, cfg.eps), p["short_conv.conv.weight"][:, 0],
                                p.get("short_conv.conv.bias"), m.short_conv.dilation, True)
    return mixed + conv


@pytest.mark.parametrize("norm,bias", [("LayerNorm", False), ("layer_norm", True), ("RMSNorm", True)])
@pytest.mark.parametrize("dtype,d,tol", [(FP, 128, 1e-5), (BF, 1024, 2e-2)])
def test_memory_layer(dev, norm, bias, dtype, d, tol):
    mem = _layer(dev, dtype, norm, bias, d)
    b, t = 2, 30
    h = torch.randn(b, t, d, device=dev).to(dtype)
    codes = torch.randint(0, 16, (b, t, mem.routes), device=dev, dtype=torch.uint8)
    out = mem.module(h, codes)
    assert not out.requires_grad
    assert om.rel_err(out.float().cpu(), _layer64(mem, h, codes)) < tol
    model = infer.memory_model(mem)
    st = infer.DecodeState.empty(model, b, t)
    outs = []
    for a, z in ((0, 1), (1, 2), (2, 9), (9, 10), (10, 30)):
        outs.append(infer.memory_step(model, 0, st, h[:, a:z].contiguous(), codes[:, a:z]))
        st.length = z
    got = torch.cat(outs, 1)
    assert not got.requires_grad and om.rel_err(got.float().cpu(), out.float().cpu()) < tol
    L = torch.full((), 5, dtype=torch.int32, device=dev)
    before = st.codes[0].clone()
    with pytest.raises(NotImplementedError, match="LayerNorm or a bias"):
        infer.static_memory_step(model, 0, st, h[:, :1], codes[:, :1], L)
    st.length = 10
    with pytest.raises(NotImplementedError, match="LayerNorm or a bias"):
        infer.tree_memory_step(model, 0, st, h[:, :2], codes[:, :2], [-1, 0])
    assert torch.equal(st.codes[0], before)


@pytest.mark.parametrize("norm,bias", [("LayerNorm", True), ("RMSNorm", True), ("LayerNorm", False)])
def test_causal_conv_module(dev, norm, bias):
    torch.manual_seed(5)
    conv = DepthwiseCausalConv(48, 4, 3, 1e-5, normalization=norm, bias=bias, zero_init=False, device=dev)
    x = torch.randn(2, 25, 48, device=dev)
    p = {k: mixing.d(v) for k, v in conv.state_dict().items()}
    want, _ = mixing.short_conv(_norm64(p, "norm", mixing.d(x), 1e-5), p["conv.weight"][:, 0], p.get("conv.bias"), 3, True)
    whole = conv(x).detach()
    assert om.rel_err(whole.cpu(), want) < 1e-5
    assert torch.equal(conv.forward_residual(x).detach(), x + whole)
    hist, ys = None, []
    for a, z in ((0, 4), (4, 5), (5, 25)):
        y, hist = conv.forward_incremental(x[:, a:z], hist)
        ys.append(y.detach())
    assert torch.equal(torch.cat(ys, 1), whole) and hist.shape == (2, 48, 9)
    with pytest.raises(ValueError, match="conv history"):
        conv.forward_incremental(x, hist[:, :, :4])
    half = conv.to(BF)                                  # fp32 rows beside parameters of another type
    p = {k: mixing.d(v) for k, v in half.state_dict().items()}
    want, _ = mixing.short_conv(_norm64(p, "norm", mixing.d(x), 1e-5), p["conv.weight"][:, 0], p.get("conv.bias"), 3, True)
    assert om.rel_err(half(x).detach().cpu(), want) < 1e-5
    conv = conv.to(FP)
    if norm == "LayerNorm":
        xl = x.clone().requires_grad_(True)
        leaves = [xl, *conv.parameters()]
        assert all(g is not None for g in torch.autograd.grad(conv(xl).sum(), leaves))


def test_the_kept_forms(dev):
    conv = DepthwiseCausalConv(64, 4, 3, 1e-5, device=dev)
    assert conv.one_kernel and isinstance(conv.norm, RMSNorm) and conv.takes_row_stats(BF)
    conv = DepthwiseCausalConv(64, 4, 3, 1e-5, normalization="LayerNorm", device=dev)
    assert not conv.one_kernel and isinstance(conv.norm, LayerNorm) and not conv.takes_row_stats(BF)
    with pytest.raises(ValueError, match="Unsupported LNGram normalization"):
        DepthwiseCausalConv(64, 4, 3, 1e-5, normalization="GroupNorm", device=dev)
