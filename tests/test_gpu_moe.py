"""The expert block (qff_rms_norm, qff_moe_gate_up, qff_moe_down) against the
definitions in 64 bits (tests/moe_ref.py), every element within the bound that
its own sums allow: fp32 sums of exact products, one rounding to the output's
type, and from 33 tokens on with 16-bit outputs fp16 operands."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _to(q):
    return None if q is None else tuple(t.to(DEV) for t in q)


def _np64(t):
    return t.detach().cpu().double().numpy()


def _ctx(**kw):
    import qff
    return qff.Context(**{"max_batch": 32, "max_ctx": 64, "max_prefill_tokens": 2048, **kw})


def _indices(rng, n, E, top, kind):
    if kind == "one":        # every pair on one expert
        return np.full((n, top), E // 2, np.int32)
    idx = rng.integers(0, E, (n, top))
    if kind == "holes":      # padded tokens, numbers that are no expert's
        bad = np.array([-1, E, -2 ** 31, 2 ** 31 - 1])
        idx = np.where(rng.random((n, top)) < 0.3, rng.choice(bad, (n, top)), idx)
        idx[n // 2] = -1
    if kind == "none":
        idx[:] = -1
    return idx.astype(np.int32)


def _weights(rng, E, D, I, sb, shared):
    q = lambda shape, cols: R.quantized(rng, shape, cols, 4, DT[sb])   # noqa: E731
    w = {"gate": q((E, I), D), "up": q((E, I), D), "down": q((E, D), I)}
    for name, shape, cols in (("shared_gate", (I,), D), ("shared_up", (I,), D), ("shared_down", (D,), I)):
        w[name] = q(shape, cols) if shared else None
    return w


def _handle(w, *names):
    import qff
    return qff.ExpertWeights(**{k: _to(v) for k, v in w.items() if not names or k in names})


# (tokens, experts, top, hidden, inter): one token, a few, one more than a tile of 16, about the border of 33, several
# tiles of an expert, more pairs than a workgroup looks through by itself; one group of columns, odd numbers of groups
# (a span's second half missing), more groups than the waves take at once
SHAPES = [(1, 8, 2, 512, 128), (1, 1, 1, 64, 64), (3, 5, 4, 192, 320), (4, 60, 8, 2048, 512), (17, 3, 2, 576, 192),
          (32, 16, 4, 512, 640), (33, 16, 4, 512, 128), (40, 2, 1, 1344, 576), (129, 60, 8, 320, 64), (300, 7, 16, 64, 1344),
          (1100, 33, 1, 128, 256)]


def _check_gate_up(ctx, w, x, idx, h_dtype, kind):
    n, top = idx.shape
    many16 = n >= 33 and h_dtype != torch.float32
    x64 = _np64(x)
    # fp16 operands: bf16 x is exact (a token's values are shifted by one power of two; what lies 2^-24 below its
    # largest is lost), fp32 x is rounded to fp16 for bf16 outputs
    x_err = np.abs(x64).max(1, keepdims=True) * 2.0 ** -37 + np.abs(x64) * (2.0 ** -11 if x.dtype == torch.float32 else 0)
    import qff
    out = torch.full((n, top + (w["shared_gate"] is not None), w["gate"][0].shape[1]), 777.0, dtype=h_dtype, device=DEV)
    got = qff.moe_gate_up(ctx, _handle(w, "gate", "up", "shared_gate", "shared_up"), x, torch.from_numpy(idx).to(DEV), out=out)
    assert got is out
    torch.cuda.synchronize()
    ref, err = R.gate_up(w["gate"], w["up"], w["shared_gate"], w["shared_up"], x64, idx, x_err if many16 else None,
                         many16 and w["gate"][1].dtype == torch.float16)
    got = _np64(got)
    hole = np.isnan(ref)
    assert (got[hole] == 777.0 if h_dtype != torch.bfloat16 else got[hole] == 776.0).all(), "rows of no expert were written"
    ok = R.within(got, np.where(hole, got, ref), np.where(hole, 0, err), h_dtype)
    assert ok.all(), f"{(~ok).sum()} of {ok.size} outside, worst {np.abs(got - ref)[~ok].max()}"
    if h_dtype == torch.float32 and not hole.all():
        d = (got - ref)[~hole]
        # 250 independent roundings of partial sums about 6 times the result's size, 2^-24 / sqrt(3) each
        assert np.linalg.norm(d) <= 4e-6 * np.linalg.norm(ref[~hole])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("x_dt,h_dt,sb,shared,kind", [("f32", "f32", "bf16", True, "any"), ("bf16", "f32", "f16", False, "holes"),
                                                      ("f32", "bf16", "f16", True, "holes"), ("bf16", "f16", "bf16", True, "one"),
                                                      ("f32", "f16", "bf16", False, "any"), ("bf16", "bf16", "f16", True, "none")])
def test_gate_up(hip, shape, x_dt, h_dt, sb, shared, kind):
    n, E, top, D, I = shape
    print(f"gate_up {shape} x={x_dt} h={h_dt} sb={sb} shared={shared} {kind}", flush=True)
    rng = np.random.default_rng(n * 1000 + E + D)
    w = _weights(rng, E, D, I, sb, shared)
    x = torch.from_numpy(rng.standard_normal((n, D))).to(DT[x_dt]).to(DEV)
    _check_gate_up(_ctx(), w, x, _indices(rng, n, E, top, kind), DT[h_dt], kind)


def _check_down(ctx, w, h, idx, y_dtype, residual, coef, rng):
    import qff
    n, top = idx.shape
    shared = w["shared_down"] is not None
    many16 = n >= 33 and y_dtype != torch.float32
    hole = (idx < 0) | (idx >= w["down"][0].shape[0])
    h = h.clone()
    h[:, :top][torch.from_numpy(hole).to(DEV)] = float("nan")   # of no expert: not read into any sum
    scores = rng.random((n, top)).astype(np.float32)
    cf = rng.random(n).astype(np.float32) if coef and shared else None
    D = w["down"][0].shape[1]
    res = torch.from_numpy(rng.standard_normal((n, D))).to(y_dtype) if residual else None
    out = res.to(DEV) if residual == "in place" else None
    got = qff.moe_down(ctx, _handle(w, "down", "shared_down"), h, torch.from_numpy(idx).to(DEV), torch.from_numpy(scores).to(DEV),
                       coef=None if cf is None else torch.from_numpy(cf).to(DEV),
                       residual=out if out is not None else None if res is None else res.to(DEV), out=out, out_dtype=y_dtype)
    torch.cuda.synchronize()
    h64 = _np64(h)
    h_err = np.abs(np.nan_to_num(h64)).max(2, keepdims=True) * 2.0 ** -37 + np.abs(h64) * (2.0 ** -11 if h.dtype == torch.float32 else 0)
    # (rows of pairs between the products and their sum have 11 bits of a block's largest entry)
    ref, err = R.down(w["down"], w["shared_down"], h64, idx, scores.astype(np.float64), None if cf is None else cf.astype(np.float64),
                      None if res is None else res.double().numpy(), h_err if many16 else None,
                      many16 and w["down"][1].dtype == torch.float16, 2.0 ** -11 if many16 else 0.0)
    got = _np64(got)
    ok = R.within(got, ref, err, y_dtype)
    assert ok.all(), f"{(~ok).sum()} of {ok.size} outside, worst {np.abs(got - ref)[~ok].max()}"
    if y_dtype == torch.float32:
        assert np.linalg.norm(got - ref) <= 4e-6 * max(np.linalg.norm(ref), 1e-30)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("h_dt,y_dt,sb,shared,kind,residual,coef", [
    ("f32", "f32", "bf16", True, "any", "in place", True), ("f16", "f32", "f16", False, "holes", "own", False),
    ("bf16", "bf16", "bf16", True, "holes", None, False), ("f16", "bf16", "bf16", True, "any", "in place", True),
    ("f32", "bf16", "f16", False, "one", "own", False), ("bf16", "f32", "f16", True, "none", None, True)])
def test_down(hip, shape, h_dt, y_dt, sb, shared, kind, residual, coef):
    n, E, top, D, I = shape
    print(f"down {shape} h={h_dt} y={y_dt} sb={sb} shared={shared} {kind} residual={residual}", flush=True)
    rng = np.random.default_rng(n * 1000 + E + I)
    w = _weights(rng, E, D, I, sb, shared)
    h = torch.from_numpy(rng.standard_normal((n, top + shared, I))).to(DT[h_dt]).to(DEV)
    _check_down(_ctx(), w, h, _indices(rng, n, E, top, kind), DT[y_dt], residual, coef, rng)


# few pairs an expert: odd numbers of groups, groups that 16-byte loads cannot take, more groups than one product's k slots
@pytest.mark.parametrize("n,E,top,D,I", [(32, 96, 8, 192, 320), (64, 200, 4, 2112, 64), (48, 128, 9, 4096, 128), (150, 300, 2, 512, 576),
                                         (32, 3, 3, 64, 64)])
@pytest.mark.parametrize("x_dt,h_dt,sb,shared,kind", [("f32", "f32", "f16", True, "holes"), ("bf16", "f16", "bf16", False, "any"),
                                                      ("f32", "bf16", "bf16", True, "one"), ("bf16", "bf16", "f16", True, "none")])
def test_few_pairs_an_expert(hip, n, E, top, D, I, x_dt, h_dt, sb, shared, kind):
    print(f"few {n} {E} {top} {D} {I} x={x_dt} h={h_dt} sb={sb} shared={shared} {kind}", flush=True)
    rng = np.random.default_rng(n + E + D)
    w = _weights(rng, E, D, I, sb, shared)
    idx = _indices(rng, n, E, top, kind)
    x = torch.from_numpy(rng.standard_normal((n, D))).to(DT[x_dt]).to(DEV)
    _check_gate_up(_ctx(), w, x, idx, DT[h_dt], kind)
    h = torch.from_numpy(rng.standard_normal((n, top + shared, I))).to(DT[h_dt]).to(DEV)
    _check_down(_ctx(), w, h, idx, DT[x_dt], "own", True, rng)


@pytest.mark.parametrize("n,y_dt", [(50, "f32"), (200, "bf16")])
def test_down_in_slices(hip, n, y_dt):
    """A context whose workspace holds the rows of a few tokens only."""
    rng = np.random.default_rng(5)
    E, top, D, I = 6, 16, 4096, 64
    w = _weights(rng, E, D, I, "bf16", True)
    h = torch.from_numpy(rng.standard_normal((n, top + 1, I))).to(DEV, DT["f16"])
    _check_down(_ctx(max_batch=n, max_prefill_tokens=1), w, h, _indices(rng, n, E, top, "holes"), DT[y_dt], "in place", True, rng)


@pytest.mark.parametrize("x_dt", ["f32", "bf16"])
def test_few_pairs_in_slices(hip, x_dt):
    """The same with few pairs an expert, on the smallest workspace that takes them."""
    rng = np.random.default_rng(6)
    n, E, top, D, I = 50, 400, 16, 2048, 64
    w = _weights(rng, E, D, I, "bf16", True)
    idx = _indices(rng, n, E, top, "holes")
    h = torch.from_numpy(rng.standard_normal((n, top + 1, I))).to(DEV, DT[x_dt])
    ctx = _ctx(max_batch=n, max_prefill_tokens=1)
    _check_down(ctx, w, h, idx, DT[x_dt], "in place", True, rng)
    _check_gate_up(ctx, w, torch.from_numpy(rng.standard_normal((n, D))).to(DEV, DT[x_dt]), idx, DT[x_dt], "holes")


def test_sizes_of_tokens(hip):
    """Every number of tokens about the borders between the forms."""
    import qff
    rng = np.random.default_rng(9)
    E, top, D, I = 4, 2, 128, 64
    w = _weights(rng, E, D, I, "bf16", True)
    ctx = _ctx()
    for n in (1, 2, 11, 12, 13, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 511, 512, 513):
        print("tokens", n, flush=True)
        x = torch.from_numpy(rng.standard_normal((n, D))).float().to(DEV)
        idx = _indices(rng, n, E, top, "holes" if n > 2 else "any")
        for dt in ("f32", "f16"):
            _check_gate_up(ctx, w, x, idx, DT[dt], "")
        h = torch.from_numpy(rng.standard_normal((n, top + 1, I))).half().to(DEV)
        for dt in ("f32", "bf16"):
            _check_down(ctx, w, h, idx, DT[dt], None, True, rng)
    # none at all
    for f in (qff.moe_gate_up(ctx, _handle(w), torch.empty(0, D, device=DEV), torch.empty(0, top, dtype=torch.int32, device=DEV)),
              qff.moe_down(ctx, _handle(w), torch.empty(0, top + 1, I, device=DEV), torch.empty(0, top, dtype=torch.int32, device=DEV),
                           torch.empty(0, top, device=DEV))):
        assert f.shape[0] == 0


def test_a_row_does_not_depend_on_the_others(hip):
    """Bit for bit: a token alone against its place among others, whatever those hold (NaN and infinity too)."""
    import qff
    rng = np.random.default_rng(3)
    E, top, D, I, n = 8, 3, 256, 128, 200
    w = _handle(_weights(rng, E, D, I, "bf16", True))
    ctx = _ctx()
    x = torch.from_numpy(rng.standard_normal((n, D))).float().to(DEV)
    idx = torch.from_numpy(_indices(rng, n, E, top, "any")).to(DEV)
    y = x.clone()
    y[::3] = float("nan")
    y[1::3] = float("inf")
    sc = torch.rand(n, top, device=DEV)
    for dt in (torch.float32, torch.bfloat16):
        a = qff.moe_gate_up(ctx, w, x, idx, out_dtype=dt)
        b = qff.moe_gate_up(ctx, w, y, idx, out_dtype=dt)
        assert torch.equal(a[2::3], b[2::3])
        # (the bf16 form's operands are fp16: rows of the same kind in both)
        c, d = a.clone(), a.clone()
        d[::3] = float("nan")
        p, q = (qff.moe_down(ctx, w, t, idx, sc, out_dtype=dt) for t in (c, d))
        keep = torch.ones(n, dtype=torch.bool, device=DEV)
        keep[::3] = False
        assert torch.equal(p[keep], q[keep])


@pytest.mark.parametrize("n", [1, 5, 32, 200, 600])
@pytest.mark.parametrize("x_dt", ["f32", "bf16"])
def test_block_together(hip, n, x_dt):
    """Norm, router, gate and up, down on the residual stream, as a layer runs them, against the same in 64 bits from
    the router's own choice."""
    import qff
    rng = np.random.default_rng(n)
    E, top, D, I = 64, 8, 512, 128
    w = _weights(rng, E, D, I, "bf16", True)
    router, gate = R.quantized(rng, (E,), D, 8, torch.bfloat16), R.quantized(rng, (1,), D, 8, torch.bfloat16)
    x = torch.from_numpy(rng.standard_normal((n, D)) * 3).float().to(DEV)
    nw = torch.from_numpy(1 + 0.1 * rng.standard_normal(D)).float().to(DEV)
    ctx, ew = _ctx(), _handle(w)
    xn, coef = qff.rms_norm(ctx, x, nw, gate=_to(gate), out_dtype=DT[x_dt])
    idx, sc, _ = qff.router_top8(ctx, *_to(router), xn)
    h = qff.moe_gate_up(ctx, ew, xn, idx)
    y = qff.moe_down(ctx, ew, h, idx, sc, coef=coef, residual=x)
    torch.cuda.synchronize()
    x64 = _np64(x)
    n64 = x64 / np.sqrt((x64 ** 2).mean(1, keepdims=True) + 1e-6) * _np64(nw)
    assert np.abs(_np64(xn) - n64).max() <= (2.0 ** -8 if x_dt == "bf16" else 2e-6) * np.abs(n64).max()
    c64 = 1 / (1 + np.exp(-(n64 @ R.dense64(gate, 8)[0])))
    assert np.abs(_np64(coef) - c64).max() <= 1e-5
    h64, _ = R.gate_up(w["gate"], w["up"], w["shared_gate"], w["shared_up"], _np64(xn), idx.cpu().numpy())
    y64, _ = R.down(w["down"], w["shared_down"], h64, idx.cpu().numpy(), _np64(sc), c64, x64)
    moe = y64 - x64
    assert np.linalg.norm(_np64(y) - y64) <= 8e-6 * np.linalg.norm(moe) + 2 ** -24 * np.linalg.norm(x64)


# ------------------------------------------------------------------------ norm

@pytest.mark.parametrize("n,cols", [(1, 2048), (3, 64), (33, 4096), (7, 8192), (1000, 2112), (5, 192)])
@pytest.mark.parametrize("x_dt,y_dt,w_dt,gate_sb", [("f32", "f32", "f32", "bf16"), ("bf16", "f32", "bf16", "f16"),
                                                    ("f32", "bf16", "f32", None), ("bf16", "bf16", "f32", "bf16")])
def test_rms_norm(hip, n, cols, x_dt, y_dt, w_dt, gate_sb):
    """Off by the sum of squares' roundings (cols / 256 + 12 at most in each thread's chain and the reduction, halved by
    the root), four more, and the output's; the coefficient's sum by cols / 256 + 16 of its terms' magnitudes."""
    import qff
    print(f"rms_norm {n}x{cols} {x_dt} {y_dt} {w_dt} gate={gate_sb}", flush=True)
    rng = np.random.default_rng(n + cols)
    x = torch.from_numpy(rng.standard_normal((n, cols)) * np.exp(rng.standard_normal((n, 1)))).to(DT[x_dt])
    x[0, :] = 0   # (eps alone)
    w = torch.from_numpy(1 + 0.1 * rng.standard_normal(cols)).to(DT[w_dt])
    gate = R.quantized(rng, (1,), cols, 8, DT[gate_sb]) if gate_sb else None
    ctx = _ctx()
    xd = x.to(DEV)
    got = qff.rms_norm(ctx, xd, w.to(DEV), 1e-6, gate=_to(gate), out_dtype=DT[y_dt])
    y, coef = got if gate else (got, None)
    x64, w64 = x.double().numpy(), w.double().numpy()
    ref = x64 / np.sqrt((x64 ** 2).mean(1, keepdims=True) + 1e-6) * w64
    err = ((cols / 256 + 12) / 2 + 6) * R.U32 * np.abs(ref)
    assert R.within(_np64(y), ref, err, DT[y_dt]).all()
    if gate:
        g = R.dense64(gate, 8)[0]
        z, mag = ref @ g, np.abs(ref) @ (np.abs(g) + 2 ** -8)
        c = 1 / (1 + np.exp(-z))
        assert (np.abs(_np64(coef) - c) <= 0.25 * (cols / 128 + 40) * R.U32 * (mag + 1) + 8 * R.U32).all()
    if x_dt == y_dt:   # in place, bit for bit the same
        again = qff.rms_norm(ctx, xd, w.to(DEV), 1e-6, gate=_to(gate), out=xd)
        assert torch.equal(again[0] if gate else again, y)


# --------------------------------------------------------- streams and graphs

def test_graphs_and_streams(hip):
    """The block captured, replayed between eager work on other inputs, each replay equal to the eager result; and
    called on another stream than the current one's inputs were made on."""
    import qff
    rng = np.random.default_rng(1)
    E, top, D, I = 16, 4, 512, 128
    w = _weights(rng, E, D, I, "bf16", True)
    ew, gate = _handle(w), _to(R.quantized(rng, (1,), D, 8, torch.bfloat16))
    nw = torch.ones(D, device=DEV)
    for n in (1, 40, 500):
        print("graph", n, flush=True)
        ctx = _ctx()
        x = torch.randn(n, D, device=DEV)
        idx = torch.from_numpy(_indices(rng, n, E, top, "any")).to(DEV)
        sc = torch.rand(n, top, device=DEV)
        bufs = [torch.empty(n, D, device=DEV), torch.empty(n, device=DEV), torch.zeros(n, top + 1, I, device=DEV, dtype=torch.float16),
                torch.empty(n, D, device=DEV)]

        def block():
            qff.rms_norm(ctx, x, nw, gate=gate, out=bufs[0], coef=bufs[1])
            qff.moe_gate_up(ctx, ew, bufs[0], idx, out=bufs[2])
            qff.moe_down(ctx, ew, bufs[2], idx, sc, coef=bufs[1], residual=x, out=bufs[3])

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            block()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            block()
        for i in range(4):
            x.copy_(torch.randn(n, D, device=DEV))
            idx.copy_(torch.from_numpy(_indices(rng, n, E, top, ["any", "holes", "one", "none"][i])).to(DEV))
            bufs[2].zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            replayed = [b.clone() for b in bufs]
            for b in bufs:
                b.fill_(3.0)
            bufs[2].zero_()
            block()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(replayed, bufs)), i
