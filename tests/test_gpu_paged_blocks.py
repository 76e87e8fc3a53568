"""Prompt slices on pages whose blocks are of 16 tokens, which the split takes
where blocks of 8 would need long chunks, and of 8 in the longest they get
(which shapes take which is checked on the host: tests/test_paged_host.py). Tolerances as in tests/test_gpu_paged_scores.py,
at scores of rms 1."""
import pytest
import torch

import paged_ref as R
from gpu_util import DEV
from test_gpu_gqa_paged import DT, Case, _randn, same_bits
from test_gpu_paged_scores import assert_near

pytestmark = pytest.mark.gpu

CONTEXT = {"max_ctx": 62000, "max_prefill_tokens": 128}
# (start, tokens): whole and partial last blocks, one block and four, cached positions that end
# inside a tile and a page, at their ends, and slices that begin there
BLOCKS_OF_16 = [(60000, 9), (59999, 16), (26000, 33), (34011, 25), (19999, 42), (14080, 64), (16001, 57)]
BLOCKS_OF_8 = [(20000, 9), (19999, 16), (8000, 33), (12011, 25), (5999, 42), (5056, 64), (6001, 57)]   # long chunks of these
TYPES = [("f32", "bf16", "f32", 16), ("bf16", "bf16", "bf16", 256), ("bf16", "f16", "bf16", 64), ("f32", "f16", "f32", 32)]


@pytest.fixture(scope="module")
def ctx():
    import qff
    c = qff.Context(max_batch=1, **CONTEXT)
    yield c
    c.close()


def _slice(start, T, page, io, kv, seed):
    """A Case whose pool page 0 is nobody's and NaN (what a bad entry is read
    as), and the slice's inputs; the slice's places hold NaN."""
    c = Case([start + T], page, io, kv, seed=seed)
    nan = torch.full_like(c.kp[:1], float("nan"))
    c.kp, c.vp = torch.cat([nan, c.kp]), torch.cat([nan, c.vp])
    c.table = torch.where(c.table >= 0, c.table + 1, c.table)
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    at, r = c.table[0].long()[pos // page], (pos % page).long()
    c.kp[at, r] = float("nan")
    c.vp[at, r] = float("nan")
    g = torch.Generator(device=DEV).manual_seed(seed)
    qg, k, v = (_randn(g, T, *s, dtype=DT[io]) for s in ((16, 512), (2, 256), (2, 256)))
    return c, qg, k, v, pos, at, r


def _check_rows(c, k, v, pos, at, r, before, kept=None):
    """The appended rows (those of `kept`), and that nothing else is written."""
    kb, vb = before
    kept = torch.ones_like(pos, dtype=torch.bool) if kept is None else kept
    want = R.rope_norm(k, c.p["k_norm_w"], pos)[kept]
    at, r = at[kept], r[kept]
    assert torch.equal(c.vp[at, r], v[kept].to(c.kv))
    step = torch.maximum(want.abs() * 2.0 ** (-7 if c.kv == torch.bfloat16 else -10), torch.full_like(want, 2.0 ** -18))
    assert ((c.kp[at, r].double() - want).abs() <= step).all()
    kb[at, r], vb[at, r] = c.kp[at, r], c.vp[at, r]
    assert same_bits(kb, c.kp) and same_bits(vb, c.vp)


def _tokens(T, kv, out):
    return min(T, 42) if (kv, out) == ("bf16", "f32") else T


@pytest.mark.parametrize("start,T", BLOCKS_OF_16 + BLOCKS_OF_8)
@pytest.mark.parametrize("io,kv,out,page", TYPES)
def test_blocks_of_16_tokens_and_long_chunks_of_8(hip, ctx, start, T, io, kv, out, page):
    import qff
    T = _tokens(T, kv, out)
    c, qg, k, v, pos, at, r = _slice(start, T, page, io, kv, seed=T)
    before = c.before()
    got = qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=DT[out])
    _check_rows(c, k, v, pos, at, r, before)
    assert_near(got, R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos), kv, 1)


@pytest.mark.parametrize("start,T,where", [(60000, 9, 0), (59999, 16, 60000), (26000, 33, 26016), (34011, 25, 34011), (19999, 42, 3000),
                                           (19999, 42, 20032), (14080, 64, 14095), (14080, 64, 14128), (14080, 64, 14143),
                                           (20000, 9, 0), (19999, 16, 20000), (8000, 33, 8016), (12011, 25, 12011), (5999, 42, 3000),
                                           (5999, 42, 6032), (5056, 64, 5071), (5056, 64, 5104), (5056, 64, 5119)])
@pytest.mark.parametrize("io,kv,out,page", [(io, kv, out, 16) for io, kv, out, _ in TYPES])
def test_pages_outside_the_pool_in_long_chunks(hip, ctx, start, T, where, io, kv, out, page):
    """The page of position `where` lies outside the pool: tokens that see it are
    NaN, those before it are right, and its rows are dropped."""
    import qff
    T = _tokens(T, kv, out)
    where = min(where, start + T - 1)
    c, qg, k, v, pos, at, r = _slice(start, T, page, io, kv, seed=where)
    table = c.table[0].clone()
    table[where // page] = c.kp.shape[0] if where % 2 else -1
    kept = pos // page != where // page
    before = c.before()
    got = qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, table, start_pos=start, out_dtype=DT[out])
    _check_rows(c, k, v, pos, at, r, before, kept)
    sees = pos >= where // page * page
    assert torch.isnan(got[sees]).all()
    if not sees.all():
        n = int((~sees).sum())
        assert_near(got[:n], R.attend(c.p, qg[:n], c.kp, c.vp, c.table[0], pos[:n]), kv, 1)


def test_value_pool_of_another_size(hip, ctx):
    """V with fewer pages than K is refused: its missing pages would be read and written."""
    import qff
    c, qg, k, v, pos, at, r = _slice(100, 9, 16, "f32", "bf16", seed=1)
    before = c.before()
    with pytest.raises(ValueError, match="k_pages and v_pages must be"):
        qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp[:-1], c.table[0], start_pos=100)
    with pytest.raises(ValueError, match="k_pages and v_pages must be"):
        qff.gqa_decode_paged(ctx, c.p, qg[:1], k[:1], v[:1], c.kp, c.vp[:-1], c.table, c.pos)
    assert same_bits(before[0], c.kp) and same_bits(before[1], c.vp)
