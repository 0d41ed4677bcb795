"""``LinearAttentionSSM`` as the token router's SSM context (whole sequences, training, decoding) against a 64-bit
restatement.

fp32 outputs are within 1e-5 (norm-relative) of 64 bits and bf16 ones within 2e-2, as the memory layer's own are;
fp32 gradients pass six sums of at most 300 roundings of 2^-24 each: 1.1e-4."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from ffnmem import infer
from ffnmem.memory.linear_attention import LinearAttentionSSM
from ffnmem.memory.wrapper import LngramMemory
from oracle import attention as oa
from oracle import memory as om
from oracle.mixing import d as to64

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


def _ssm(dev, d=128, n=48, dtype=FP, heads=4, key_dim=16, kv_heads=2, seed=0):
    torch.manual_seed(seed)
    m = LinearAttentionSSM(d, n, heads, key_dim, kv_heads)
    with torch.no_grad():                            # weights of a trained size: every term of the output counts
        m.w_qkv.weight.normal_(0, d ** -0.5)
        m.w_g.weight.normal_(0, d ** -0.5)
        for norm in (m.norm, m.out_norm):
            norm.weight.normal_(1, 0.2)
            norm.bias.normal_(0, 0.2)
    return m.to(dtype).to(dev)


def _params(m) -> dict:
    return {k: to64(v) for k, v in m.named_parameters()}


def _restated(p: dict, m, emb, lengths=None, state=None):
    b, t = emb.shape[:2]
    x = F.layer_norm(emb, emb.shape[-1:], p["norm.weight"], p["norm.bias"], m.norm.eps)
    hq, hk, dk, dv = m.heads, m.kv_heads, m.key_dim, m.value_dim
    q, k, v = F.linear(x, p["w_qkv.weight"]).split((hq * dk, hk * dk, hk * dv), -1)
    g = F.logsigmoid(F.linear(x, p["w_g.weight"]) + p["decay_bias"])
    y, end = oa.linear_attention(q.unflatten(-1, (hq, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hk, dv)), g, dk ** -0.5,
                                 state, lengths)
    z = F.group_norm(y.reshape(b * t, m.state_dim), hq, p["out_norm.weight"], p["out_norm.bias"], m.out_norm.eps)
    y = F.silu(z).view(b, t, m.state_dim)
    if lengths is not None:
        y = y * (torch.arange(t)[None] < lengths[:, None])[..., None]
    return y, end


def test_forward_and_gradients(dev):
    m = _ssm(dev)
    gen = torch.Generator().manual_seed(3)
    emb, dy = torch.randn(3, 50, 128, generator=gen), torch.randn(3, 50, 48, generator=gen)
    lengths = torch.tensor([50, 20, 0], dtype=torch.int32)
    e = emb.to(dev).requires_grad_(True)
    y, end = m(e, lengths=lengths.to(dev), return_state=True)
    with torch.no_grad():
        assert torch.equal(m(e, lengths=lengths.to(dev)), y)
    p = {k: v.requires_grad_(True) for k, v in _params(m).items()}
    e64 = emb.double().requires_grad_(True)
    want, wend = _restated(p, m, e64, lengths)
    assert om.rel_err(y.detach().cpu(), want.detach()) < 1e-5 and om.rel_err(end.detach().cpu(), wend.detach()) < 1e-5
    assert (y[2] == 0).all() and (y[1, 20:] == 0).all()
    names = list(p)
    got = torch.autograd.grad(y, [e, *(dict(m.named_parameters())[k] for k in names)], dy.to(dev))
    ref = torch.autograd.grad(want, [e64, *(p[k] for k in names)], dy.double())
    for k, a, b in zip(["emb", *names], got, ref):
        assert om.rel_err(a.cpu(), b) < 1.1e-4, k


def test_what_stands_behind_a_sequence_has_no_part(dev):
    m = _ssm(dev)
    own = torch.tensor([30, 4], device=dev)
    emb = torch.randn(2, 30, 128, device=dev)
    dirty = emb.clone()
    dirty[1, 4:] = float("nan")
    outs = []
    for e in (emb, dirty):
        e = e.requires_grad_(True)
        y, end = m(e, lengths=own, return_state=True)
        outs.append([y.detach(), end.detach(), *torch.autograd.grad(y.sum() + end.sum(), [*m.parameters(), e])])
    assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("dtype,tol", [(FP, 1e-5), (BF, 2e-2)])
def test_parts_and_steps_continue_a_sequence(dev, dtype, tol):
    m = _ssm(dev, dtype=dtype)
    emb = torch.randn(2, 90, 128, generator=torch.Generator().manual_seed(4)).to(dtype).to(dev)
    with torch.no_grad():
        whole, end = m(emb, return_state=True)
        y, st = m(emb[:, :17], return_state=True)
        ys, kept = [y], st.clone()
        y2, st2 = m(emb[:, 17:80], state=st, return_state=True)
        assert torch.equal(st, kept)                     # the given state stays: a way back
        ys.append(y2)
        for i in range(80, 90):
            y, st2 = m.step(st2, emb[:, i])
            ys.append(y[:, None])
        one, _ = m.step(None, emb[:, 0])
    assert om.rel_err(torch.cat(ys, 1).float().cpu(), whole.float().cpu()) < tol
    assert om.rel_err(one.float().cpu(), whole[:, 0].float().cpu()) < tol
    assert om.rel_err(st2.cpu(), end.cpu()) < tol
    want, _ = _restated(_params(m), m, to64(emb))
    assert om.rel_err(whole.float().cpu(), want) < tol


@pytest.mark.parametrize("d,n,heads,key_dim", [(72, 21, 3, 7), (100, 30, 5, 33)])
def test_bf16_training_of_odd_widths(dev, d, n, heads, key_dim):
    m = _ssm(dev, d, n, BF, heads, key_dim, 1)
    emb = torch.randn(2, 40, d, device=dev).to(BF)
    own = torch.tensor([40, 7], device=dev)
    y, end = m(emb, lengths=own, return_state=True)
    assert y.dtype == BF and end.dtype == FP and bool((y[1, 7:] == 0).all())
    (y.float().sum() + end.sum()).backward()
    for k, p in m.named_parameters():
        assert p.grad.shape == p.shape and p.grad.dtype == BF and bool(torch.isfinite(p.grad).all()), k


def test_no_tokens_and_no_sequences(dev):
    m = _ssm(dev)
    emb = torch.randn(2, 5, 128, device=dev)
    with torch.no_grad():
        _, state = m(emb, return_state=True)
        y, after = m(emb[:, :0], state=state, return_state=True)
        assert y.shape == (2, 0, 48) and torch.equal(after, state)
        assert m(emb[:0]).shape == (0, 5, 48)
    y, after = m(emb[:, :0], state=state, return_state=True)
    grads = torch.autograd.grad(y.sum() + after.sum(), list(m.parameters()), allow_unused=True)
    assert all(g is None or bool((g == 0).all()) for g in grads)


def test_training_step_captured(dev):
    """Forward and backward of the block replayed from a graph, against eager steps in between."""
    m = _ssm(dev, dtype=BF)
    emb = torch.randn(2, 70, 128, device=dev).to(BF)
    params = list(m.parameters())

    def step():
        y = m(emb)
        return [y.detach(), *torch.autograd.grad(y.float().square().sum(), params)]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        emb.copy_(torch.randn(2, 70, 128, device=dev))
        ref = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # the features and the block's own kernels give equal bits; torch's products of the gradients are deterministic too
        assert all(torch.equal(p, q) for p, q in zip(out, ref)), rep


def test_step_replayed_from_a_graph(dev):
    m = _ssm(dev, dtype=BF)
    emb = torch.randn(4, 128, device=dev).to(BF)
    state = m.empty_state(4)

    def step():
        y, new = m.step(state, emb)
        state.copy_(new)
        return y

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    ref_state = None
    state.zero_()
    for rep in range(4):
        emb.copy_(torch.randn(4, 128, device=dev))
        ref, ref_state = m.step(ref_state, emb)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(state, ref_state), rep


def test_context_of_the_token_router(dev):
    """The memory layer routed by the features: a whole sequence at once, and decoded token by token with the
    features, the code cache and the conv cache moving on together."""
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
        state, outs = None, []
        for i in range(t):
            f, state = ssm.step(state, table[tok[:, i]])
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
        with pytest.raises(NotImplementedError, match="LinearAttentionSSM"):
            fn()
