"""qff_sample against the definition row by row in 64 bits (tests/moe_ref.py):
tokens equal, chances to fp32's rounding. Weights are whole numbers, so borders
are exact: rows of equal logits put every border on a tie."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV

pytestmark = pytest.mark.gpu


def _run(ctx, logits, u, **kw):
    import qff
    dt = {"temperature": torch.float32, "top_k": torch.int32, "top_p": torch.float32, "min_p": torch.float32}
    args = {k: torch.tensor(v, dtype=dt[k], device=DEV) for k, v in kw.items() if v is not None}
    tok, prob = qff.sample(ctx, logits, torch.tensor(u, dtype=torch.float32, device=DEV), **args)
    torch.cuda.synchronize()
    return tok.cpu().numpy(), prob.cpu().numpy()


def _check(ctx, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    tok, prob = _run(ctx, logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    rows = logits.float().cpu().numpy()
    for b in range(rows.shape[0]):
        at = lambda v, d: d if v is None else v[b]   # noqa: E731
        ref = R.sample_row(rows[b], u[b], at(temperature, 1.0), at(top_k, 0), at(top_p, 1.0), at(min_p, 0.0))
        assert tok[b] == ref[0], (b, tok[b], ref)
        assert abs(prob[b] - ref[1]) <= 2 ** -23 * ref[1], (b, prob[b], ref)


def _ctx(n=32):
    import qff
    return qff.Context(max_batch=n, max_ctx=64, max_prefill_tokens=1)


@pytest.mark.parametrize("vocab,batch", [(1, 3), (2, 2), (63, 4), (500, 8), (4099, 32), (20000, 5), (151936, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_filters(hip, vocab, batch, dtype):
    print("sample", vocab, batch, dtype, flush=True)
    ctx = _ctx()
    rng = np.random.default_rng(vocab)
    B = batch
    for case in range(6):
        logits = torch.from_numpy(rng.standard_normal((B, vocab)) * rng.choice([0.5, 2, 6])).to(dtype).to(DEV)
        u = rng.random(B)
        kw = {}
        if case in (1, 4, 5):
            kw["top_k"] = rng.integers(1, min(vocab, 300) + 1, B).tolist()
        if case in (2, 4, 5):
            kw["top_p"] = rng.uniform(0.05, 1.0, B).tolist()
        if case in (3, 5):
            kw["min_p"] = rng.uniform(0.001, 0.5, B).tolist()
        if case:
            kw["temperature"] = rng.uniform(0.3, 2.0, B).tolist()
        _check(ctx, logits, u.tolist(), **kw)


def test_ties_and_borders(hip):
    """Equal logits: every border lies on a tie, broken by index."""
    ctx = _ctx()
    V = 1000
    flat = torch.zeros(8, V, device=DEV)
    u = [0.0, 0.25, 0.5, 0.75, 0.999, 0.5, 1.0, -1.0]
    _check(ctx, flat, u)
    _check(ctx, flat, u, top_p=[0.5, 0.25, 0.125, 0.001, 1e-30, 0.999, 0.75, 0.5])
    _check(ctx, flat, u, top_k=[1, 2, 10, 999, 1000, 1001, 2 ** 31 - 1, -5])
    _check(ctx, flat, u, top_k=[7] * 8, top_p=[0.5] * 8, min_p=[1.0] * 8)
    two = flat.clone()
    two[:, 3::7] = 2.0    # a group of equal largest ones, -0 among the others
    two[:, 5::7] = -0.0
    _check(ctx, two, u, top_p=[0.9, 0.5, 0.3, 0.6, 0.7, 0.99, 0.1, 0.95])
    _check(ctx, two, u, top_k=[3, 143, 144, 200, 500, 10, 142, 1])
    _check(ctx, two, u, top_k=[150] * 8, top_p=[0.2, 0.5, 0.9, 0.95, 0.99, 0.999, 0.01, 0.7], temperature=[0.1, 5, 1, 100, 1e30, 1, 1e-30, 2])


@pytest.mark.parametrize("vocab", [15872, 15873, 40000, 262144])
def test_ties_of_a_whole_row(hip, vocab):
    """More equal logits at a border than the last launch keeps in LDS, alone and beside larger and smaller ones."""
    print("ties", vocab, flush=True)
    ctx = _ctx()
    rows = torch.zeros(6, vocab, device=DEV)
    rows[1, ::3] = 0.25            # two values
    rows[2, vocab // 2] = 3.0      # one ahead of the rest
    rows[3, ::2] = -float("inf")
    rows[4] = torch.arange(vocab, device=DEV) % 5 * 1e-3   # five values close together, all in the border's bin or not
    rows[5, -1] = -20.0
    u = [0.0, 0.3, 0.999, 0.5, 0.75, 1.0]
    _check(ctx, rows, u, top_k=[1, vocab // 2, vocab - 1, 17, vocab // 3, vocab])
    _check(ctx, rows, u, top_p=[0.5, 0.9, 0.1, 0.999, 0.3, 0.25])
    _check(ctx, rows.bfloat16(), u, temperature=[0.7] * 6, top_k=[vocab // 2] * 6, top_p=[0.5] * 6, min_p=[0.0, 0.9, 0.0, 0.5, 0.99, 0.1])


def test_greedy_and_odd_settings(hip):
    ctx = _ctx()
    inf, nan = float("inf"), float("nan")
    l = torch.randn(8, 3001, device=DEV)
    l[0, 100] = l[0, 2900] = 50.0
    l[1] = -inf
    l[2] = nan
    l[3, 7] = nan
    l[4, :] = -inf
    l[4, 1234] = -3.0
    l[5, 17] = l[5, 2000] = inf
    l[6, 1:] = -inf
    u = [0.1, 0.5, 0.5, 0.9, 0.9, 0.7, 0.3, 0.999999]
    _check(ctx, l, u)
    _check(ctx, l, u, temperature=[0.0, 0.0, 0.0, -1.0, nan, 0.0, 0.0, 0.0])
    _check(ctx, l, u, top_k=[5] * 8, top_p=[0.9] * 8, min_p=[0.01] * 8)
    _check(ctx, l, u, top_p=[0.0, -1.0, 0.5, nan, 2.0, 0.5, 0.5, 0.0])
    _check(ctx, l, u, min_p=[2.0, 1.0, 0.5, nan, -1.0, 0.5, 1.0, 1.0])
    tok, _ = _run(ctx, l, [nan] * 8)
    assert tok[4] == 1234 and tok[1] == -1


def test_spread_of_draws(hip):
    """Every u of a grid falls where the running sum says: all tokens of a short row are reached."""
    ctx = _ctx(64)
    l = torch.tensor([0.0, -1.0, -2.0, 1.0, -40.0, 0.5], device=DEV).repeat(64, 1)
    u = ((np.arange(64) + 0.5) / 64).tolist()
    _check(ctx, l, u)
    tok, _ = _run(ctx, l, u)
    assert set(tok.tolist()) == {0, 1, 2, 3, 5} and (np.diff(tok) >= 0).all()


def test_graph_replays(hip):
    import qff
    ctx = _ctx()
    l = torch.randn(4, 5000, device=DEV)
    u = torch.rand(4, device=DEV)
    k = torch.tensor([0, 10, 50, 0], dtype=torch.int32, device=DEV)
    p = torch.tensor([1.0, 0.9, 1.0, 0.5], device=DEV)
    out, prob = torch.empty(4, dtype=torch.int32, device=DEV), torch.empty(4, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        qff.sample(ctx, l, u, top_k=k, top_p=p, out=out, prob=prob)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        qff.sample(ctx, l, u, top_k=k, top_p=p, out=out, prob=prob)
    for i in range(4):
        l.copy_(torch.randn(4, 5000, device=DEV) * (i + 1))
        u.copy_(torch.rand(4, device=DEV))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        a, b = out.clone(), prob.clone()
        c, d = qff.sample(ctx, l, u, top_k=k, top_p=p)
        torch.cuda.synchronize()
        assert torch.equal(a, c) and torch.equal(b, d)
