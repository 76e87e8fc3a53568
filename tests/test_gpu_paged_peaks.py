"""The paged calls on rows whose softmax is rescaled on the way (planted K rows,
tests/paged_peaks.py): within a tile, from tile to tile, between the waves that
share a row's positions, and between chunks; some rows of a wave only, and scores
that reach the last step before a maximum is raised (fp16 weights of up to 2^15).
tests/test_paged_peaks.py says what mistakes they would show.

Tolerances as in tests/test_gpu_paged_scores.py, with the largest score (about
63) in place of the scores' rms: both errors are proportional to the scores."""
import random

import pytest
import torch

import paged_peaks as P
import paged_ref as R
from gpu_util import DEV
from test_gpu_gqa_paged import DT, Case, _groups, _randn
from test_gpu_paged_scores import assert_near

pytestmark = pytest.mark.gpu

S = P.MOST / P.LOG2E
TYPES = [("f32", "bf16", "f32"), ("bf16", "bf16", "bf16"), ("f32", "f16", "f32"), ("bf16", "f16", "bf16")]


@pytest.fixture(scope="module")
def ctx():
    import qff
    c = qff.Context(max_batch=32, max_ctx=46080, max_prefill_tokens=128)
    yield c
    c.close()


def _check(c, out, kv, seqs=None):
    for b in seqs or range(c.B):
        assert_near(out[b], R.attend(c.p, c.qg[b:b + 1], c.kp, c.vp, c.table[b], c.pos[b:b + 1])[0], kv, S, b)


@pytest.mark.parametrize("lengths", [[130, 700, 66, 4096, 2049], [33, 64, 18], [200] * 20, [40000]])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_decode_rescaled(hip, ctx, io, kv, out, lengths):
    import qff
    c, rng = Case(lengths, 16, io, kv, seed=len(lengths)), random.Random(len(lengths))
    for b, n in enumerate(lengths):
        P.plant(c, [b], 0, n - 1, rng)
        c.k[b, 1] = c.qg[b, 11, :256]      # the new token's own row is one head's peak
    _check(c, qff.gqa_decode_paged(ctx, *c.args(), out_dtype=DT[out]), kv)


@pytest.mark.parametrize("sizes,prefix", [([2, 5, 8, 3], [900, 1500, 3000, 128]), ([16, 7], [2000, 700])])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_shared_decode_rescaled(hip, ctx, io, kv, out, sizes, prefix):
    """Blocks of 2 to 8 sequences, single ones behind them."""
    import qff
    c, group, shared = _groups(sizes, prefix, [1, 40, 300, 7], 64, io=io, kv=kv, seed=len(sizes))
    rng, first = random.Random(3), 0
    for m in sizes:
        lead = int(shared[first])
        P.plant(c, list(range(first, first + m)), 0, lead, rng, part=0.5 if lead > 400 * m else 0.2)
        for b in range(first, first + m):
            P.plant(c, [b], lead, c.lengths[b] - 1, rng, each=3)
        first += m
    _check(c, qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=DT[out]), kv)


@pytest.mark.parametrize("io,kv,out", TYPES)
def test_shared_decode_rescaled_large_blocks(hip, ctx, io, kv, out):
    """28 sequences over 45000 positions: blocks of 9 to 16, long chunks."""
    import qff
    c, group, shared = _groups([16, 12], [45000, 44000], [1, 90, 700], 64, io=io, kv=kv, seed=8)
    rng = random.Random(4)
    for first, m in ((0, 16), (16, 12)):
        lead = int(shared[first])
        P.plant(c, list(range(first, first + m)), 0, lead, rng, each=12)
        for b in range(first, first + m):
            P.plant(c, [b], lead, c.lengths[b] - 1, rng, each=3)
    _check(c, qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=DT[out]), kv, seqs=(0, 1, 7, 15, 16, 21, 27))


@pytest.mark.parametrize("start,T", [(700, 5), (130, 8), (1000, 40), (0, 42), (64, 17), (8000, 33), (20000, 9), (5999, 42), (26000, 33), (19999, 42)])
@pytest.mark.parametrize("io,kv,out", TYPES)
def test_short_slices_rescaled(hip, ctx, io, kv, out, start, T):
    """Blocks of 8 and 16 tokens; the slice's own k rows are peaks of the tokens
    from there on, at their own position first."""
    import qff
    c, rng = Case([start + T], 16, io, kv, seed=T), random.Random(T)
    g = torch.Generator(device=DEV).manual_seed(T)
    qg, k, v = (_randn(g, T, *shape, dtype=DT[io]) for shape in ((16, 512), (2, 256), (2, 256)))
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    q = R.rope_norm(qg[:, :, :256], c.p["q_norm_w"], pos)
    P.plant(c, [0], 0, start, rng, q=q, part=0.5 if start > 100 * T else 0.1)
    for i in range(0, T, 3):
        k[i, i % 2] = qg[i, 8 * (i % 2) + i % 8, :256]
    got = qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=DT[out])
    assert_near(got, R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos), kv, S)


@pytest.mark.parametrize("start,T", [(3000, 130), (900, 300)])
@pytest.mark.parametrize("io,kv,out", [t for t in TYPES if t[2] == "bf16"])
def test_long_slices_rescaled(hip, ctx, io, kv, out, start, T):
    """The fp16-operand kernels on pages give the flat call's bits on such rows too."""
    import qff
    n = -(-(start + T) // 16)
    c, rng = Case([start + T], 16, io, kv, seed=T), random.Random(T)
    small = qff.Context(max_batch=1, max_ctx=4096, max_prefill_tokens=512)
    g = torch.Generator(device=DEV).manual_seed(T)
    qg, k, v = (_randn(g, T, *shape, dtype=DT[io]) for shape in ((16, 512), (2, 256), (2, 256)))
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    P.plant(c, [0], 0, start, rng, q=R.rope_norm(qg[:8, :, :256], c.p["q_norm_w"], pos[:8]))
    at = c.table[0, :n].long()
    kc, vc = c.kp[at].flatten(0, 1).contiguous(), c.vp[at].flatten(0, 1).contiguous()
    ref = qff.gqa_prefill(small, c.p, qg, k, v, kc, vc, start_pos=start, out_dtype=DT[out])
    got = qff.gqa_prefill_paged(small, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=DT[out])
    assert not torch.isnan(got).any() and torch.equal(got, ref)
    small.close()
