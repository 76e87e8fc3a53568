"""The paged calls at scores other than those of unit normals, against the
64-bit restatement (tests/paged_ref.py).

Tolerances, for scores of rms s (norm weights of about s, unit normal K):
  fp32 outputs   5e-6 s of the row's 2-norm. A score is summed in 24 MFMA steps whose
                 partial sums are about 3 s: off by sqrt(24) 3 s 2^-24 = 9e-7 s, a row by
                 sqrt(2) of it; four times that.
  bf16 outputs   half a step, 2^-8 of the value, and c s of the row's rms: c = 12
                 sqrt(2) e, where e s is a score's rms error and 12 the largest of
                 10^6 products of two normals. An fp16 cache's q has two terms (2^-22),
                 so e is the sums' 9e-7, c = 1.5e-5, the bar 2e-5. A bf16
                 cache's q is off by half of 2^-17 of itself at most, 2^-18 / sqrt(3) =
                 2.2e-6 rms, c = 3.7e-5, the bar 4e-5. (One fp16 term: e = 2.8e-4,
                 thirty times the bar of any s.)"""
import pytest
import torch

import paged_ref as R
from gpu_util import DEV
from test_gpu_gqa_paged import DT, Case, _groups, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import qff
    c = qff.Context(max_batch=32, max_ctx=4096, max_prefill_tokens=128)
    yield c
    c.close()


def assert_near(out, ref, kv, s, what=""):
    err = (out.double() - ref).abs()
    assert not torch.isnan(err).any(), what
    if out.dtype == torch.float32:
        rel = float((err.norm(dim=-1) / ref.norm(dim=-1)).max())
        assert rel <= 5e-6 * s, (what, rel)
    else:
        rms = ref.square().mean(-1, keepdim=True).sqrt()
        bar = 2.0 ** -8 * ref.abs() + (2e-5 if kv == "f16" else 4e-5) * s * rms
        assert (err <= bar).all(), (what, float(((err - bar) / rms).max()))


TYPES = [("bf16", "f16", "bf16"), ("f32", "f16", "bf16"), ("bf16", "bf16", "bf16"), ("f32", "f16", "f32"), ("f32", "bf16", "f32")]


@pytest.mark.parametrize("s", [1, 8])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_decode_at_score_magnitudes(hip, ctx, io, kv, out, s):
    import qff
    c = Case([1, 50, 700, 2048, 4000], 32, io, kv, seed=s)
    c.p["q_norm_w"] *= s
    got = qff.gqa_decode_paged(ctx, *c.args(), out_dtype=DT[out])
    for b in range(c.B):
        assert_near(got[b], R.attend(c.p, c.qg[b:b + 1], c.kp, c.vp, c.table[b], c.pos[b:b + 1])[0], kv, s, b)


@pytest.mark.parametrize("s", [1, 8])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_shared_decode_at_score_magnitudes(hip, ctx, io, kv, out, s):
    import qff
    c, group, shared = _groups([2, 12, 1, 8, 3], [900, 2000, 30, 1100, 3000], [1, 40, 300], 64, io=io, kv=kv, seed=s)
    c.p["q_norm_w"] *= s
    got = qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=DT[out])
    for b in range(c.B):
        assert_near(got[b], R.attend(c.p, c.qg[b:b + 1], c.kp, c.vp, c.table[b], c.pos[b:b + 1])[0], kv, s, b)


@pytest.mark.parametrize("s", [1, 8])
@pytest.mark.parametrize("start,T", [(0, 5), (1500, 8), (700, 40), (3500, 42)])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_short_slices_at_score_magnitudes(hip, ctx, io, kv, out, start, T, s):
    import qff
    c = Case([start + T], 16, io, kv, seed=T)
    c.p["q_norm_w"] *= s
    g = torch.Generator(device=DEV).manual_seed(T)
    qg, k, v = (_randn(g, T, *shape, dtype=DT[io]) for shape in ((16, 512), (2, 256), (2, 256)))
    got = qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=DT[out])
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    assert_near(got, R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos), kv, s)


@pytest.mark.parametrize("max_ctx,start,T", [(512, 448, 64), (512, 470, 42), (200, 130, 64), (100, 41, 42), (100, 3, 9), (64, 62, 2)])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_short_slices_in_contexts_of_few_partials(hip, io, kv, out, max_ctx, start, T):
    """A slice's precision depends on its tokens and types, not on how many
    partial rows its context has: one to three chunks a token here."""
    import qff
    if T * (3 if (kv, out) == ("bf16", "f32") else 2) > 128:
        T = 42
    small = qff.Context(max_batch=1, max_ctx=max_ctx, max_prefill_tokens=64)
    c = Case([start + T], 16, io, kv, seed=T)
    g = torch.Generator(device=DEV).manual_seed(T)
    qg, k, v = (_randn(g, T, *shape, dtype=DT[io]) for shape in ((16, 512), (2, 256), (2, 256)))
    got = qff.gqa_prefill_paged(small, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=DT[out])
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    assert_near(got, R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos), kv, 1)
    small.close()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_a_row_without_a_value_leaves_the_others(hip, ctx, io, kv, out, bad):
    """q, and the gate, of single sequences or tokens NaN or infinite, next to
    others in a wave, a block and a row block: those keep their bits."""
    import qff
    c, group, shared = _groups([2, 12, 1, 8, 3], [900, 2000, 30, 1100, 3000], [1, 40, 300], 64, io=io, kv=kv, seed=5)
    start = [t.clone() for t in (c.kp, c.vp)]
    rows, gates = [0, 3, 9, 14, 17, 25], [1, 5]
    for call, more in ((qff.gqa_decode_paged, ()), (qff.gqa_decode_shared, (group, shared))):
        c.kp.copy_(start[0])
        c.vp.copy_(start[1])
        want = call(ctx, *c.args(), *more, out_dtype=DT[out])
        qg = c.qg.clone()
        for i, b in enumerate(rows):
            qg[b, (5 * i) % 16, 31 * i] = bad
        for b in gates:
            qg[b, 2, 300] = float("nan")
        c.kp.copy_(start[0])
        c.vp.copy_(start[1])
        got = call(ctx, c.p, qg, *c.args()[2:], *more, out_dtype=DT[out])
        for i, b in enumerate(rows):
            assert torch.isnan(got[b, (5 * i) % 16]).all()
            want[b, (5 * i) % 16] = got[b, (5 * i) % 16] = 0
        for b in gates:
            assert torch.isnan(got[b, 2, 44])
            want[b, 2, 44] = got[b, 2, 44] = 0
        assert torch.equal(got, want)
    T = 40
    c = Case([700 + T], 16, io, kv, seed=T)
    qg, k, v = (_randn(torch.Generator(device=DEV).manual_seed(T), T, *s, dtype=DT[io]) for s in ((16, 512), (2, 256), (2, 256)))
    run = lambda q: qff.gqa_prefill_paged(ctx, c.p, q, k, v, c.kp, c.vp, c.table[0], start_pos=700, out_dtype=DT[out])   # noqa: E731
    want, other = run(qg), qg.clone()
    for t in (0, 7, 8, 39):
        other[t, t % 16, t] = bad
    got = run(other)
    for t in (0, 7, 8, 39):
        assert torch.isnan(got[t, t % 16]).all()
        want[t, t % 16] = got[t, t % 16] = 0
    assert torch.equal(got, want)
