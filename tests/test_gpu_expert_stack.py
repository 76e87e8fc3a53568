"""A stack whose layers have expert blocks, and its next tokens: each block against
64 bits from the kernels' own layer input and the router's own choice
(tests/moe_ref.py), and a captured step against the eager one."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV
from qff import synth

pytestmark = pytest.mark.gpu
E, I, VOCAB, B = 24, 128, 1000, 5


def _np64(t):
    return t.detach().cpu().double().numpy()


@pytest.fixture(scope="module")
def model(hip):
    import qff
    from qff import stack as S
    g = torch.Generator(device=DEV).manual_seed(21)
    dnp = {k: torch.from_numpy(v).to(DEV) for k, v in synth.deltanet_params().items()}
    gqp = {k: torch.from_numpy(v).to(DEV) for k, v in synth.gqa_params().items()}
    layers = S.random_layers(4, g, dnp, gqp, device=DEV)
    for L in layers:
        L["mlp"] = S.random_mlp(E, I, g, device=DEV)
        L["mlp"]["norm_w"] = 1 + 0.1 * torch.randn(2048, device=DEV, generator=g)
    head = {"norm_w": 1 + 0.1 * torch.randn(2048, device=DEV, generator=g), "lm_head": S.random_q4(VOCAB, 2048, g, DEV)}
    ctx = qff.Context(max_batch=8, max_ctx=256, max_prefill_tokens=64)
    yield ctx, layers, head
    ctx.close()


def _stack(model, mlp=True, pages=False, head=True):
    from qff.pages import PageTable
    from qff.stack import AttentionStack
    ctx, layers, hd = model
    layers = layers if mlp else [{k: v for k, v in L.items() if k != "mlp"} for L in layers]
    table = PageTable(40, 16, B, 256, device=DEV) if pages else None
    return AttentionStack(ctx, layers, B, 256, pages=table, head=hd if head else None)


def _block64(M, x):
    """The block's update of x from the router's own choice on the kernels' norm."""
    import qff
    ctx = qff.Context(max_batch=64, max_ctx=64, max_prefill_tokens=64)
    xn, coef = qff.rms_norm(ctx, x, M["norm_w"], gate=M["gate"])
    idx, sc, _ = qff.router_top8(ctx, *M["router"], xn)
    torch.cuda.synchronize()
    host = [tuple(t.cpu() for t in q) for q in M["experts"].matrices]
    h, _ = R.gate_up(host[0], host[1], host[3], host[4], _np64(xn), idx.cpu().numpy())
    y, _ = R.down(host[2], host[5], h, idx.cpu().numpy(), _np64(sc), _np64(coef), _np64(x))
    ctx.close()
    return y - _np64(x)


def test_decode_layers(model):
    """Layer by layer: the same layer without its block, then the block in 64 bits."""
    st, bare = _stack(model), _stack(model, mlp=False)
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(B, 2048, device=DEV, generator=g)
    for step in range(2):
        pos = torch.full((B,), step, dtype=torch.int32, device=DEV)
        for l, L in enumerate(st.layers):
            y = x.clone()
            bare.layer_step(l, y, pos)
            st.layer_step(l, x, pos)
            torch.cuda.synchronize()
            moe = _block64(L["mlp"], y)
            # as in the block's own test: sums to 8e-6 of what the block adds, and the residual's rounding
            assert np.linalg.norm(_np64(x) - _np64(y) - moe) <= 8e-6 * np.linalg.norm(moe) + 2 ** -23 * np.linalg.norm(_np64(y))
            x.div_(x.pow(2).mean(1, keepdim=True).sqrt())


def test_prefill_is_the_layers_on_a_slice(model):
    st, bare = _stack(model, pages=True), _stack(model, mlp=False, pages=True)
    g = torch.Generator(device=DEV).manual_seed(6)
    x0 = torch.randn(40, 2048, device=DEV, generator=g)
    one = _stack(model, pages=True)
    one.layers, one.kinds, one.states = st.layers[:1], st.kinds[:1], one.states[:1]
    bare.layers, bare.kinds, bare.states = bare.layers[:1], bare.kinds[:1], bare.states[:1]
    x, y = x0.clone(), x0.clone()
    one.prefill(2, x)
    bare.prefill(2, y)
    torch.cuda.synchronize()
    moe = _block64(st.layers[0]["mlp"], y)
    assert np.linalg.norm(_np64(x) - _np64(y) - moe) <= 8e-6 * np.linalg.norm(moe) + 2 ** -23 * np.linalg.norm(_np64(y))
    st.prefill(2, x0)   # (all layers run)
    assert torch.isfinite(x0).all()


def test_next_tokens(model):
    from qff import ops
    st = _stack(model)
    ctx, _, head = model
    g = torch.Generator(device=DEV).manual_seed(8)
    for n in (1, B):
        x = torch.randn(n, 2048, device=DEV, generator=g)
        u = torch.rand(n, device=DEV, generator=g)
        k = torch.full((n,), 20, dtype=torch.int32, device=DEV)
        p = torch.full((n,), 0.9, device=DEV)
        tok, chance = st.next_tokens(x, u, top_k=k, top_p=p)
        logits = ops.q4_norm_matmul_parts(ctx, [head["lm_head"]], x, head["norm_w"], st.eps)[0]
        torch.cuda.synchronize()
        for b in range(n):
            ref = R.sample_row(logits[b].cpu().numpy(), float(u[b]), 1.0, 20, float(p[b]), 0.0)
            assert int(tok[b]) == ref[0] and abs(float(chance[b]) - ref[1]) <= 2 ** -23 * ref[1]


def test_captured_step_and_tokens(model):
    """A step and its next tokens in a graph, replayed with eager steps of another stack between."""
    st, eager = _stack(model), _stack(model)
    g = torch.Generator(device=DEV).manual_seed(9)
    x, u = torch.zeros(B, 2048, device=DEV), torch.zeros(B, device=DEV)
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    st.decode_step(x, pos)
    st.next_tokens(x, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st.decode_step(x, pos)
        st.next_tokens(x, u)
    for S in st.states:
        for t in S.values():
            t.zero_()
    for step in range(4):
        xin = torch.randn(B, 2048, device=DEV, generator=g)
        x.copy_(xin)
        u.copy_(torch.rand(B, device=DEV, generator=g))
        pos.fill_(step)
        y = xin.clone()
        eager.decode_step(y, pos)
        tok, chance = eager.next_tokens(y, u)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, y) and torch.equal(st.tokens, tok) and torch.equal(st.chances, chance)
