"""The expert block in forms and sizes that tests/test_gpu_moe.py leaves out: large tiles of more than 32 groups of
columns, calls that take their tokens in several slices, the shapes of a stack's own prompts, outputs of very different
size side by side, and rows of very small and very large values."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV
from test_gpu_moe import DT, _check_down, _check_gate_up, _ctx, _handle, _indices, _np64, _to, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [2112, 4096])
@pytest.mark.parametrize("in_dt,out_dt,sb", [("f32", "f32", "f16"), ("bf16", "f16", "bf16"), ("f32", "bf16", "f16")])
def test_large_tiles_of_many_groups(hip, cols, in_dt, out_dt, sb):
    """More than 32 groups: the constant parts' terms come in several rounds."""
    print(f"many groups {cols} {in_dt} {out_dt} {sb}", flush=True)
    rng = np.random.default_rng(cols)
    n, E, top = 130, 3, 2
    ctx = _ctx()
    w = _weights(rng, E, cols, 64, sb, True)
    x = torch.from_numpy(rng.standard_normal((n, cols))).to(DT[in_dt]).to(DEV)
    _check_gate_up(ctx, w, x, _indices(rng, n, E, top, "holes"), DT[out_dt], "holes")
    w = _weights(rng, E, 128, cols, sb, True)
    for h_dt in {in_dt, "f16"}:
        h = torch.from_numpy(rng.standard_normal((n, top + 1, cols))).to(DT[h_dt]).to(DEV)
        _check_down(ctx, w, h, _indices(rng, n, E, top, "holes"), DT["bf16" if out_dt == "bf16" else "f32"], "own", True, rng)


def test_gate_up_in_slices(hip):
    """fp32 rows of x whose two terms exceed the workspace: 1024 tokens, then 476."""
    rng = np.random.default_rng(4)
    n, E, top, D, I = 1500, 4, 2, 4096, 64
    w = _weights(rng, E, D, I, "bf16", True)
    x = torch.from_numpy(rng.standard_normal((n, D))).float().to(DEV)
    _check_gate_up(_ctx(), w, x, _indices(rng, n, E, top, "holes"), DT["f32"], "holes")


@pytest.mark.parametrize("n", [100, 300])
@pytest.mark.parametrize("x_dt,h_dt,y_dt", [("f32", "f32", "f32"), ("bf16", "f16", "bf16")])
def test_prompts_of_a_stack(hip, n, x_dt, h_dt, y_dt):
    """hidden 2048 and inter 512 in large tiles, fp32 throughout as the stack's prompts are, and in 16 bits."""
    print(f"prompt {n} {x_dt} {h_dt} {y_dt}", flush=True)
    rng = np.random.default_rng(n)
    E, top, D, I = 8, 4, 2048, 512
    w = _weights(rng, E, D, I, "bf16", True)
    idx = _indices(rng, n, E, top, "any")
    ctx = _ctx()
    _check_gate_up(ctx, w, torch.from_numpy(rng.standard_normal((n, D))).to(DT[x_dt]).to(DEV), idx, DT[h_dt], "any")
    h = torch.from_numpy(rng.standard_normal((n, top + 1, I))).to(DT[h_dt]).to(DEV)
    _check_down(ctx, w, h, idx, DT[y_dt], "in place", True, rng)


@pytest.mark.parametrize("h_dt,n", [("f16", 210), ("f32", 210), ("f16", 40)])
def test_a_large_output_beside_small_ones(hip, h_dt, n):
    """bf16 outputs of which one in each 64 is a thousand times the others (whose weights are small, so that every constant
    part stays below 8): a pair's rows between the products and their
    sum hold 11 bits of each value, not of the largest beside it (2^-39 of that)."""
    rng = np.random.default_rng(11)
    E, top, D, I = 3, 6, 192, 128
    w = _weights(rng, E, D, I, "bf16", False)["down"]
    big = torch.zeros(D, dtype=torch.bool)
    big[5::64] = True
    for t in w[1:]:
        t[:, ~big] /= 1024
    import qff
    idx = _indices(rng, n, E, top, "any")
    h = torch.from_numpy(rng.standard_normal((n, top, I))).to(DT[h_dt])
    sc = rng.random((n, top)).astype(np.float32)
    got = _np64(qff.moe_down(_ctx(), qff.ExpertWeights(down=_to(w)), h.to(DEV), torch.from_numpy(idx).to(DEV), torch.from_numpy(sc).to(DEV),
                             out_dtype=torch.bfloat16))
    h64 = h.double().numpy()
    h_err = np.abs(h64) * (2.0 ** -11 if h_dt == "f32" else 0) + np.abs(h64).max(2, keepdims=True) * 2.0 ** -37
    ref, err = R.down(w, None, h64, idx, sc.astype(np.float64), None, None, h_err)
    for m in range(n):
        for j in range(top):
            p = np.abs(R.dense64([t[idx[m, j]] for t in w]) @ h64[m, j])
            err[m] += sc[m, j] * (2.0 ** -11 * p + 2.0 ** -39 * p.max())
    small = ~big.numpy()
    for part in (small, ~small):
        ok = R.within(got[:, part], ref[:, part], err[:, part], torch.bfloat16)
        assert ok.all(), f"{(~ok).sum()} of {ok.size} outside"


@pytest.mark.parametrize("n,E,top", [(2, 3, 2), (70, 200, 4), (210, 3, 1)])
@pytest.mark.parametrize("x_dt", ["f32", "bf16", "f16"])
def test_rows_of_any_size(hip, n, E, top, x_dt):
    """Rows between 2^-90 and 2^90 (fp16: down to its last bit) beside each other, each to its own size."""
    import qff
    rng = np.random.default_rng(n)
    D, I = 128, 192
    w = _weights(rng, E, D, I, "bf16", False)
    idx = _indices(rng, n, E, top, "any")
    lo, hi = (-90, 90) if x_dt != "f16" else (-24, 14)
    h = torch.from_numpy(rng.standard_normal((n, top, I)) * 2.0 ** rng.integers(lo, hi, (n, top, 1))).to(DT[x_dt])
    h64 = h.double().numpy()
    for y_dt in ("f32", "bf16"):
        got = _np64(qff.moe_down(_ctx(), _handle(w, "down"), h.to(DEV), torch.from_numpy(idx).to(DEV), torch.ones(n, top, device=DEV),
                                 out_dtype=DT[y_dt]))
        few = n < 33 or y_dt == "f32"
        h_err = np.abs(h64) * (2.0 ** -22 if few else 2.0 ** -11) * (x_dt == "f32") + np.abs(h64).max(2, keepdims=True) * 2.0 ** -37
        ref, err = R.down(w["down"], None, h64, idx, np.ones((n, top)), None, None, h_err, part=0.0 if few else 2.0 ** -11)
        ok = R.within(got, ref, err, DT[y_dt])
        assert ok.all(), f"{y_dt}: {(~ok).sum()} of {ok.size} outside"
    if x_dt == "f16":
        return
    # gate and up, silu(g) u: rows up to 2^40 keep the product inside fp32
    x = torch.from_numpy(rng.standard_normal((n, D)) * 2.0 ** rng.integers(-60, 40, (n, 1))).to(DT[x_dt])
    x64 = x.double().numpy()
    x_err = np.abs(x64) * 2.0 ** -22 + np.abs(x64).max(1, keepdims=True) * 2.0 ** -37
    got = _np64(qff.moe_gate_up(_ctx(), _handle(w, "gate", "up"), x.to(DEV), torch.from_numpy(idx).to(DEV)))
    with np.errstate(over="ignore"):
        ref, err = R.gate_up(w["gate"], w["up"], None, None, x64, idx, x_err)
    # (what lies below 2^-120, where fp32's smallest numbers end, is held to 2^-149)
    assert (np.abs(got - ref) <= err * (1 + R.U32) + R.U32 * np.abs(ref) + 2.0 ** -148).all()


def test_rms_norm_of_more_rows_than_a_grid(hip):
    """2^24 + 5 rows: a launch holds 2^24 - 1 (2^32 work-items, 256 a row). Rows on both sides of the border equal those
    of a call of their own."""
    import qff
    n, cols, ctx = 2 ** 24 + 5, 64, _ctx()
    x = torch.randn(2 ** 16, cols, device=DEV).bfloat16().repeat(n // 2 ** 16 + 1, 1)[:n]
    w = 1 + 0.1 * torch.randn(cols, device=DEV)
    gate = _to(R.quantized(np.random.default_rng(0), (1,), cols, 8, torch.bfloat16))
    y, coef = torch.full_like(x, 7.0), torch.full((n,), 7.0, device=DEV)
    qff.rms_norm(ctx, x, w, gate=gate, out=y, coef=coef)
    for a, b in ((0, 64), (2 ** 24 - 40, n)):
        ref = qff.rms_norm(ctx, x[a:b], w, gate=gate)
        assert torch.equal(y[a:b], ref[0]) and torch.equal(coef[a:b], ref[1])
    assert torch.equal(y[:2 ** 16], y[2 ** 23:2 ** 23 + 2 ** 16])


def test_most_experts_and_slots(hip):
    """512 experts, 16 a token and a shared one, in small and large tiles."""
    rng = np.random.default_rng(12)
    E, top, D, I = 512, 16, 128, 64
    w = _weights(rng, E, D, I, "f16", True)
    ctx = _ctx()
    for n, dt in ((40, "f32"), (300, "f32"), (600, "bf16")):
        print("512 experts", n, flush=True)
        idx = _indices(rng, n, E, top, "holes")
        x = torch.from_numpy(rng.standard_normal((n, D))).to(DEV, DT[dt])
        _check_gate_up(ctx, w, x, idx, DT[dt], "holes")
        h = torch.from_numpy(rng.standard_normal((n, top + 1, I))).to(DEV, DT[dt])
        _check_down(ctx, w, h, idx, DT[dt], "in place", True, rng)


def test_more_tokens_than_a_grid_has_rows(hip):
    """66000 tokens: slices of at most 65535. The last slice's tokens against a call of their own, the others by parts."""
    import qff
    rng = np.random.default_rng(13)
    n, E, top, D, I = 66000, 4, 2, 64, 64
    w = _handle(_weights(rng, E, D, I, "bf16", True))
    ctx = _ctx(max_batch=1, max_prefill_tokens=n)
    x = torch.randn(n, D, device=DEV)
    idx = torch.randint(-1, E + 1, (n, top), dtype=torch.int32, device=DEV)
    sc = torch.rand(n, top, device=DEV)
    h = qff.moe_gate_up(ctx, w, x, idx, out=torch.zeros(n, top + 1, I, device=DEV))
    y = qff.moe_down(ctx, w, h, idx, sc, residual=x)
    torch.cuda.synchronize()
    for a, b in ((0, 1000), (65000, n), (65535, n)):
        g = qff.moe_gate_up(ctx, w, x[a:b], idx[a:b].contiguous(), out=torch.zeros(b - a, top + 1, I, device=DEV))
        z = qff.moe_down(ctx, w, h[a:b], idx[a:b].contiguous(), sc[a:b].contiguous(), residual=x[a:b])
        # (the same exact products; a call's form decides their order: 20 roundings of sums a few times the results)
        assert (g - h[a:b]).norm() <= 1e-6 * g.norm() and (z - y[a:b]).norm() <= 1e-6 * z.norm()
    ctx.close()
