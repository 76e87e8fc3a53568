"""GPU parity of the paged full-attention calls (qff_gqa_decode_paged,
qff_gqa_decode_shared, qff_gqa_prefill_paged) against a 64-bit restatement
(tests/paged_ref.py).

The attention is checked over the cache as the call left it, after the
appended rows have been checked by themselves (the v entries bit for bit, the k
entries to one ulp of the cache's type or 2^-18: a value beside a rounding
border may round either way), so a rounding that falls the other way is not
counted twice.

Tolerances. fp32 outputs: a score is a sum of 256 products taken in 24 steps
(8 MFMA steps of three terms), |partial sums| about 3, so its error is about
sqrt(24) 3 2^-24 = 9e-7, that of a softmax weight sqrt(2) of it, and an output
row's, relative to its 2-norm, the same: 1.3e-6; the bar is four times that,
5e-6. bf16 outputs: half a step, 2^-8 of the value, and for a bf16 cache 1e-4
of the row's rms for the scores' two-term q and weights (2^-16 each). For an
fp16 cache q and the weights are one fp16 term, off by half a step of 2^-11
relative, 2^-11 / sqrt(3) = 2.8e-4 rms: a score (terms of rms 1 in sum) by as
much, a weight by as much again, so an output by sqrt(2) 2.8e-4 = 4e-4 of the
row's rms. What a row of few positions is off by is the product of two normal
values, the error that all its dims share and a dim's own spread of v: the
largest of 10^6 such products is z times their rms with sqrt(2 / (pi z)) e^-z =
10^-6, z = 12: 4.8e-3, the bar 5e-3.
Prefill: slices of more than 128 tokens take the launches of qff_gqa_prefill
after the pages are gathered, so the same bits; of tokens x terms <= 128 the
decode's kernels and tolerances; those between, fp16 operands: 3e-4 of the row
(four times it here)."""
import numpy as np
import pytest
import torch

import paged_ref as R
from gpu_util import DEV

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _params(g):
    return {k: 1 + 0.1 * torch.randn(256, device=DEV, generator=g) for k in ("q_norm_w", "k_norm_w")}


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def same_bits(a, b) -> bool:
    """Whether two 16-bit tensors hold the same bits (NaN as NaN)."""
    return bool((a.view(torch.int16) == b.view(torch.int16)).all())


class Case:
    """A batch of sequences of `lengths` positions (0: a padded slot), the last
    of them the new token's, in a pool whose rows hold NaN wherever no
    sequence's cached position lies. share: per sequence the sequence whose
    first `common` positions' pages it holds (itself: none)."""

    def __init__(self, lengths, page, io="f32", kv="bf16", seed=0, share=None, common=None, spare=3, cols=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rng = np.random.default_rng(seed)
        B = len(lengths)
        self.B, self.page, self.lengths, self.kv = B, page, list(lengths), DT[kv]
        need = [-(-n // page) for n in lengths]
        self.cols = cols or max(max(need), 1)
        own = list(need)
        for b in range(B):
            if share and share[b] != b:
                own[b] = need[b] - common[b] // page
        total = sum(own) + spare
        order = rng.permutation(total)
        table = np.full((B, self.cols), -7, np.int32)   # entries past a sequence's last are not read
        at = 0
        for b in range(B):
            have = need[b] - own[b]
            if have:
                table[b, :have] = table[share[b], :have]
            table[b, have:need[b]] = order[at:at + own[b]]
            at += own[b]
        self.table_np = table
        self.table = torch.from_numpy(table).to(DEV)
        self.p = _params(g)
        io = DT[io]
        self.qg, self.k, self.v = _randn(g, B, 16, 512, dtype=io), _randn(g, B, 2, 256, dtype=io), _randn(g, B, 2, 256, dtype=io)
        self.kp = torch.full((total, page, 2, 256), float("nan"), dtype=self.kv, device=DEV)
        self.vp = self.kp.clone()
        for b, n in enumerate(lengths):
            if n > 1:
                i = torch.arange(n - 1, device=DEV)
                at = self.table[b].long()[i // page]
                lead = i < (common[b] if share and share[b] != b else 0)   # (the leader wrote those)
                kr, vr = _randn(g, n - 1, 2, 256, dtype=self.kv), _randn(g, n - 1, 2, 256, dtype=self.kv)
                self.kp[at[~lead], (i % page)[~lead]] = kr[~lead]
                self.vp[at[~lead], (i % page)[~lead]] = vr[~lead]
        self.pos = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device=DEV)

    def args(self):
        return (self.p, self.qg, self.k, self.v, self.kp, self.vp, self.table, self.pos)

    def expected_row(self, b):
        """What the appended k and v rows round to."""
        k = R.rope_norm(self.k[b:b + 1], self.p["k_norm_w"], self.pos[b:b + 1])[0]
        return k, self.v[b].to(self.kv)

    def check(self, out, before, seqs=None):
        """`before`: (k pool, v pool) ahead of the call; outputs of the
        sequences `seqs` (all)."""
        kb, vb = before
        for b in range(self.B):
            n = self.lengths[b]
            if n == 0:
                assert torch.isnan(out[b]).all()
                continue
            at, r = int(self.table_np[b, (n - 1) // self.page]), (n - 1) % self.page
            k, v = self.expected_row(b)
            assert torch.equal(self.vp[at, r], v), b
            step = torch.maximum(k.abs() * 2.0 ** (-7 if self.kv == torch.bfloat16 else -10), torch.full_like(k, 2.0 ** -18))
            assert ((self.kp[at, r].double() - k).abs() <= step).all(), b
            kb[at, r], vb[at, r] = self.kp[at, r], self.vp[at, r]
            if seqs is not None and b not in seqs:
                continue
            ref = R.attend(self.p, self.qg[b:b + 1], self.kp, self.vp, self.table[b], self.pos[b:b + 1])[0]
            assert_near(out[b], ref, b, self.kv)
        assert same_bits(kb, self.kp)   # nothing else is written
        assert same_bits(vb, self.vp)

    def before(self):
        return self.kp.clone(), self.vp.clone()


def assert_near(out, ref, what="", kv=torch.bfloat16, fp16_operands=False):
    err = (out.double() - ref).abs()
    assert not torch.isnan(err).any(), what
    if out.dtype == torch.float32:
        rel = (err.norm(dim=-1) / ref.norm(dim=-1)).max()
        assert rel <= (1.2e-3 if fp16_operands else 5e-6), (what, float(rel))
    else:
        rms = ref.square().mean(-1, keepdim=True).sqrt()
        rest = 5e-3 if kv == torch.float16 or fp16_operands else 1e-4
        over = (err - (2.0 ** -8 * ref.abs() + rest * rms)).max()
        assert over <= 0, (what, float(over))


@pytest.fixture(scope="module")
def ctx():
    import qff
    c = qff.Context(max_batch=80, max_ctx=4096, max_prefill_tokens=1024)
    yield c
    c.close()


EDGES = [1, 2, 15, 16, 17, 0, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 2048]


# --------------------------------------------------------------------- decode

@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("io,kv,out", [("f32", "bf16", "f32"), ("bf16", "bf16", "bf16"), ("f32", "f16", "f32"),
                                       ("bf16", "f16", "f32"), ("f32", "bf16", "bf16")])
def test_decode_paged_edges(hip, ctx, page, io, kv, out):
    """Lengths around tiles, chunks and pages, a padded slot among them, in
    one batch; everything no sequence holds is NaN."""
    import qff
    c = Case(EDGES, page, io, kv, seed=page)
    before = c.before()
    c.check(qff.gqa_decode_paged(ctx, *c.args(), out_dtype=DT[out]), before)


@pytest.mark.parametrize("n", [1, 2, 40, 700, 4095, 4096])
def test_decode_paged_one_sequence(hip, ctx, n):
    import qff
    c = Case([n], 32, seed=n)
    before = c.before()
    c.check(qff.gqa_decode_paged(ctx, *c.args(), out_dtype=torch.float32), before)


def test_decode_paged_large_batch(hip, ctx):
    """More sequences than a wave has lanes, ragged."""
    import qff
    rng = np.random.default_rng(5)
    c = Case([int(n) for n in rng.integers(0, 900, 80)], 16, "bf16", "f16", seed=9)
    before = c.before()
    c.check(qff.gqa_decode_paged(ctx, *c.args(), out_dtype=torch.bfloat16), before)


def test_decode_paged_long_chunks(hip):
    """16 sequences of 64K in pages of 16: chunks of more pages than a wave
    holds table entries at once."""
    import qff
    big = qff.Context(max_batch=16, max_ctx=65536, max_prefill_tokens=1)
    c = Case([65536 - 37 * b for b in range(16)], 16, "bf16", "bf16", seed=3)
    before = c.before()
    c.check(qff.gqa_decode_paged(big, *c.args(), out_dtype=torch.float32), before, seqs=(0, 7, 15))
    big.close()


def test_decode_paged_pool_past_4_gib(hip, ctx):
    """Pages behind byte 2^32 of a pool."""
    import qff
    c = Case([700, 65, 1], 64, seed=21)
    far = 70_000
    kp = torch.empty(far + c.kp.shape[0], 64, 2, 256, dtype=torch.bfloat16, device=DEV)
    vp = torch.empty_like(kp)
    kp[far:], vp[far:] = c.kp, c.vp
    table = torch.where(c.table >= 0, c.table + far, c.table)
    ref = qff.gqa_decode_paged(ctx, *c.args(), out_dtype=torch.float32)
    out = qff.gqa_decode_paged(ctx, c.p, c.qg, c.k, c.v, kp, vp, table, c.pos, out_dtype=torch.float32)
    assert torch.equal(out, ref)
    assert same_bits(kp[far:], c.kp)
    assert same_bits(vp[far:], c.vp)


@pytest.mark.parametrize("shared", [False, True])
def test_decode_pages_outside_the_pool(hip, ctx, shared):
    """A table entry outside the pool makes its sequence NaN (the shared
    prefix's: every sequence that reads it), and touches nothing else; an
    append to such a page is dropped."""
    import qff
    share, common = ([0, 0, 0, 3, 4], [0, 256, 256, 0, 0]) if shared else (None, None)
    c = Case([300, 310, 320, 129, 200], 64, seed=2, share=share, common=common)
    c.table[3, 1] = c.kp.shape[0]      # in the middle
    c.table[4, 3] = -1                 # the page the new token goes to
    nan = {3, 4}
    if shared:
        c.table[0, 2] = 1 << 30        # shared by 0, 1 and 2 through row 0
        nan |= {0, 1, 2}
    kb, vb = c.before()
    if shared:
        group = torch.tensor([5, 5, 5, -1, -1], dtype=torch.int32, device=DEV)
        out = qff.gqa_decode_shared(ctx, *c.args(), group, torch.full_like(group, 256), out_dtype=torch.float32)
    else:
        out = qff.gqa_decode_paged(ctx, *c.args(), out_dtype=torch.float32)
    for b, n in enumerate(c.lengths):
        assert torch.isnan(out[b]).all() == (b in nan), b
        if b not in nan:
            assert_near(out[b], R.attend(c.p, c.qg[b:b + 1], c.kp, c.vp, c.table[b], c.pos[b:b + 1])[0])
        if b != 4:
            at, r = int(c.table_np[b, (n - 1) // 64]), (n - 1) % 64
            kb[at, r], vb[at, r] = c.kp[at, r], c.vp[at, r]
    assert same_bits(kb, c.kp)
    assert same_bits(vb, c.vp)


# --------------------------------------------------------------------- shared

def _groups(sizes, prefix, tails, page, **kw):
    """Groups of `sizes` sequences holding the same `prefix[g]` positions (the
    whole pages of them; the rest of the last page copied, as a fork does)."""
    share, common, lengths, group, shared = [], [], [], [], []
    at = 0
    for g, (m, S) in enumerate(zip(sizes, prefix)):
        for i in range(m):
            share.append(at)
            common.append(S // page * page if i else 0)
            lengths.append(S + tails[(at + i) % len(tails)])
            group.append(g if m > 1 else -1)
            shared.append(S // page * page)
        at += m
    c = Case(lengths, page, share=share, common=common, **kw)
    dev = dict(dtype=torch.int32, device=DEV)
    return c, torch.tensor(group, **dev), torch.tensor(shared, **dev)


@pytest.mark.parametrize("io,kv,out", [("f32", "bf16", "f32"), ("bf16", "bf16", "bf16"), ("bf16", "f16", "bf16"),
                                       ("f32", "f16", "f32"), ("bf16", "bf16", "f32"), ("f32", "bf16", "bf16")])
@pytest.mark.parametrize("page", [16, 128])
def test_decode_shared_groups(hip, ctx, page, io, kv, out):
    """Groups of 1, 2, 3, 5, 8, 9 and 16 sequences, prefixes from less than a
    tile to several chunks, tails of one token on."""
    import qff
    c, group, shared = _groups([2, 1, 3, 5, 9, 16, 8], [1000, 300, 130, 2048, 700, 1500, 40], [1, 2, 17, 200, 33], page,
                               io=io, kv=kv, seed=page)
    before = c.before()
    c.check(qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=DT[out]), before)


@pytest.mark.parametrize("sizes", [[17], [33, 4], [40, 40], [7, 64, 3]])
def test_decode_shared_large_groups(hip, ctx, sizes):
    """Groups cut into blocks of 16, and across the 64th sequence."""
    import qff
    c, group, shared = _groups(sizes, [900] * len(sizes), [1, 40, 5], 32, io="bf16", seed=len(sizes))
    before = c.before()
    c.check(qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=torch.float32), before)


def test_decode_shared_any_lengths(hip, ctx):
    """shared_len negative, past a member's position, no multiple of 16 or of
    the page; a padded slot in the middle of a group; the same values under two
    numbers. Only the common positions may be read together."""
    import qff
    c, group, shared = _groups([6, 5], [640, 512], [1, 30, 100], 64, seed=4)
    c.lengths[3] = 0
    c.pos[3] = -1
    for k, s in enumerate([5000, 333, 640, 77, 640, 640, -4, 512, 512, 512, 512]):
        shared[k] = s
    before = c.before()
    c.check(qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=torch.float32), before)
    # a member whose own position lies inside what the others share
    c, group, shared = _groups([5], [640], [1, 30], 64, seed=5)
    c.lengths[2] = 200
    c.pos[2] = 199
    c.table[2, :4] = torch.tensor([int(x) for x in c.table_np[2, :3]] + [int(c.table_np[2, 10])], dtype=torch.int32)
    c.table_np = c.table.cpu().numpy()
    # (its fourth page is its own: a fork's copy of the shared one)
    c.kp[c.table[2, 3].long()] = c.kp[c.table[0, 3].long()]
    c.vp[c.table[2, 3].long()] = c.vp[c.table[0, 3].long()]
    before = c.before()
    c.check(qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=torch.float32), before)


def test_decode_shared_without_groups_and_with_one_sequence(hip, ctx):
    import qff
    c = Case(EDGES, 16, seed=8)
    before = c.before()
    none = torch.full((c.B,), -1, dtype=torch.int32, device=DEV)
    c.check(qff.gqa_decode_shared(ctx, *c.args(), none, c.pos, out_dtype=torch.float32), before)
    c = Case([500], 16, seed=8)
    before = c.before()
    c.check(qff.gqa_decode_shared(ctx, *c.args(), none[:1] + 1, c.pos, out_dtype=torch.float32), before)


def test_decode_shared_long_prefix(hip):
    """A prefix of 128K in pages of 16: prefix chunks of more pages than a
    wave holds table entries at once."""
    import qff
    big = qff.Context(max_batch=8, max_ctx=140_000, max_prefill_tokens=1)
    c, group, shared = _groups([3], [131072 + 48], [1, 700, 90], 16, io="bf16", seed=6)
    before = c.before()
    c.check(qff.gqa_decode_shared(big, *c.args(), group, shared, out_dtype=torch.float32), before)
    big.close()


@pytest.mark.parametrize("kv,out", [("f16", "bf16"), ("bf16", "bf16")])
def test_decode_shared_large_blocks_long_chunks(hip, kv, out):
    """Four groups of 16 over 36000 positions in pages of 16: a large block's
    chunks of more pages than a wave holds table entries at once, and what
    follows each prefix in chunks of its own."""
    import qff
    big = qff.Context(max_batch=64, max_ctx=40_000, max_prefill_tokens=1)
    c, group, shared = _groups([16] * 4, [36000, 35984, 36000 - 16 * 7, 33333], [1, 700, 90, 2000], 16, io="bf16", kv=kv, seed=16)
    before = c.before()
    c.check(qff.gqa_decode_shared(big, *c.args(), group, shared, out_dtype=DT[out]), before, seqs=(0, 13, 16, 33, 47, 63))
    big.close()


@pytest.mark.parametrize("kv,out", [("f16", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("where", [0, 9, 14])
def test_decode_shared_large_blocks_pages_outside_the_pool(hip, ctx, kv, out, where):
    """A bad entry in the prefix of a group of 12 (at its start, inside, in its
    last tile): the sequence that names it is NaN, and so may be those of its group
    that are read through its row; no other is wrong."""
    import qff
    c, group, shared = _groups([12, 11], [960, 960], [1, 70, 5], 64, io="bf16", kv=kv, seed=where)
    c.table[0, where] = c.kp.shape[0] + 5
    out = qff.gqa_decode_shared(ctx, *c.args(), group, shared, out_dtype=DT[out])
    assert torch.isnan(out[0]).all()
    for b in range(1, 23):
        if b < 12 and torch.isnan(out[b]).all():
            continue
        assert_near(out[b], R.attend(c.p, c.qg[b:b + 1], c.kp, c.vp, c.table[b], c.pos[b:b + 1])[0], b, c.kv)
    assert not torch.isnan(out[12:]).any()


@pytest.mark.parametrize("kv,out", [("f16", "bf16"), ("bf16", "f32")])
def test_decode_shared_long_blocks_pages_outside_the_pool(hip, kv, out):
    """The same in a prefix whose chunks are long: bad entries in two groups of
    three, near each end of their prefixes."""
    import qff
    big = qff.Context(max_batch=64, max_ctx=40_000, max_prefill_tokens=1)
    c, group, shared = _groups([16, 13, 16], [33000, 36000, 35000], [1, 70, 300], 64, io="bf16", kv=kv, seed=7)
    c.table[0, 1] = -1
    c.table[16, 561] = c.kp.shape[0]
    out = qff.gqa_decode_shared(big, *c.args(), group, shared, out_dtype=DT[out])
    assert torch.isnan(out[0]).all() and torch.isnan(out[16]).all()
    for b in (1, 15, 17, 28, 29, 44):
        if b < 29 and torch.isnan(out[b]).all():
            continue
        assert_near(out[b], R.attend(c.p, c.qg[b:b + 1], c.kp, c.vp, c.table[b], c.pos[b:b + 1])[0], b, c.kv)
    assert not torch.isnan(out[29:]).any()
    big.close()


# --------------------------------------------------------- graphs and streams

@pytest.mark.parametrize("shared", [False, True])
def test_decode_captured(hip, ctx, shared):
    """A captured step replayed while the positions move on, eager work
    between the replays: every replay as the eager call."""
    import qff
    c, group, shared_len = _groups([4, 2], [300, 200], [3, 9, 60], 64, seed=12)
    more = (group, shared_len) if shared else ()
    call = qff.gqa_decode_shared if shared else qff.gqa_decode_paged
    out = torch.empty(c.B, 16, 256, device=DEV)
    start = [t.clone() for t in (c.kp, c.vp, c.pos)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(ctx, *c.args(), *more, out=out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ctx, *c.args(), *more, out=out)
    for t, x in zip((c.kp, c.vp, c.pos), start):
        t.copy_(x)
    kp, vp = start[0].clone(), start[1].clone()
    eager = torch.empty_like(out)
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        call(ctx, c.p, c.qg, c.k, c.v, kp, vp, c.table, c.pos, *more, out=eager)
        assert torch.equal(out, eager), step
        assert same_bits(kp, c.kp)
        assert same_bits(vp, c.vp)
        c.pos += 1
        c.qg.normal_()
        c.k.normal_()


def test_calls_on_a_side_stream(hip, ctx):
    import qff
    c, group, shared = _groups([5], [400], [7, 50], 64, seed=13)
    ref = qff.gqa_decode_shared(ctx, *c.args(), group, shared)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = qff.gqa_decode_shared(ctx, *c.args(), group, shared)
    s.synchronize()
    assert torch.equal(out, ref)


# -------------------------------------------------------------------- prefill

@pytest.mark.parametrize("start,T", [(0, 129), (0, 700), (5, 130), (63, 192), (2011, 300), (3000, 1024)])
@pytest.mark.parametrize("io,kv,out,page", [("f32", "bf16", "bf16", 16), ("bf16", "f16", "f32", 64), ("bf16", "bf16", "bf16", 256),
                                            ("f32", "f16", "bf16", 32)])
def test_prefill_paged_is_the_flat_one(hip, ctx, start, T, io, kv, out, page):
    """Pages gathered: the bits of qff_gqa_prefill, rows and caches, whatever
    the pool holds elsewhere."""
    import qff
    g = torch.Generator(device=DEV).manual_seed(start + T)
    n = -(-(start + T) // page)
    total = n + 4
    table = torch.randperm(total, device=DEV, generator=g)[:n].to(torch.int32)
    p, kv, io = _params(g), DT[kv], DT[io]
    qg, k, v = _randn(g, T, 16, 512, dtype=io), _randn(g, T, 2, 256, dtype=io), _randn(g, T, 2, 256, dtype=io)
    kc, vc = (torch.full((n * page, 2, 256), float("nan"), dtype=kv, device=DEV) for _ in range(2))
    kc[:start], vc[:start] = _randn(g, start, 2, 256, dtype=kv), _randn(g, start, 2, 256, dtype=kv)
    kp, vp = (torch.full((total, page, 2, 256), float("nan"), dtype=kv, device=DEV) for _ in range(2))
    kp[table.long()], vp[table.long()] = kc.view(n, page, 2, 256), vc.view(n, page, 2, 256)
    row = torch.cat([table, torch.full((3,), -1, dtype=torch.int32, device=DEV)]) if (n + 3) * page <= 4096 else table
    ref = qff.gqa_prefill(ctx, p, qg, k, v, kc, vc, start_pos=start, out_dtype=DT[out])
    got = qff.gqa_prefill_paged(ctx, p, qg, k, v, kp, vp, row, start_pos=start, out_dtype=DT[out])
    assert not torch.isnan(got).any()
    assert torch.equal(got, ref)
    for pool, flat in ((kp, kc), (vp, vc)):
        want = torch.full_like(pool, float("nan"))
        want[table.long()] = flat.view(n, page, 2, 256)
        assert same_bits(pool, want)


@pytest.mark.parametrize("start,T", [(0, 1), (0, 2), (0, 8), (60, 8), (125, 5), (1021, 7), (2047, 3), (3000, 4), (4088, 8), (0, 9), (0, 17), (0, 128), (1, 1), (15, 1), (63, 2), (64, 33), (900, 33), (897, 16),
                                     (2000, 5), (2000, 42), (2000, 43), (3000, 64), (3000, 65), (3000, 100), (3968, 128),
                                     (4095, 1)])
@pytest.mark.parametrize("io,kv,out,page", [("f32", "bf16", "f32", 16), ("bf16", "f16", "bf16", 64), ("bf16", "bf16", "bf16", 256),
                                            ("f32", "f16", "f32", 32)])
def test_prefill_paged_short(hip, ctx, start, T, io, kv, out, page):
    """Short slices: blocks of 16 tokens and less, chunks that begin past a
    token's own position, pages that end inside a tile, NaN in every row that
    holds no position."""
    import qff
    c = Case([start + T], page, io, kv, seed=start + T)
    g = torch.Generator(device=DEV).manual_seed(T)
    qg, k, v = (_randn(g, T, *s, dtype=DT[io]) for s in ((16, 512), (2, 256), (2, 256)))
    for i in range(start, start + T):   # (Case wrote what precedes its last position)
        at = int(c.table_np[0, i // page])
        c.kp[at, i % page] = float("nan")
        c.vp[at, i % page] = float("nan")
    kb, vb = c.before()
    got = qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=DT[out])
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    want_k = R.rope_norm(k, c.p["k_norm_w"], pos)
    at, r = c.table[0].long()[pos // page], (pos % page).long()
    assert torch.equal(c.vp[at, r], v.to(c.kv))
    step = torch.maximum(want_k.abs() * 2.0 ** (-7 if c.kv == torch.bfloat16 else -10), torch.full_like(want_k, 2.0 ** -18))
    assert ((c.kp[at, r].double() - want_k).abs() <= step).all()
    terms = {("bf16", "f32"): 3, ("f16", "bf16"): 1}.get((kv, out), 2)
    assert_near(got, R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos), "", c.kv, fp16_operands=T * terms > 128)
    kb[at, r], vb[at, r] = c.kp[at, r], c.vp[at, r]
    assert same_bits(kb, c.kp) and same_bits(vb, c.vp)


@pytest.mark.parametrize("kv,out", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "bf16")])
def test_prefill_paged_short_in_a_small_context(hip, kv, out):
    """A context whose partial rows hold few chunks."""
    import qff
    small = qff.Context(max_batch=1, max_ctx=2048, max_prefill_tokens=64)
    c = Case([1900], 16, "f32", kv, seed=3)
    g = torch.Generator(device=DEV).manual_seed(3)
    qg, k, v = _randn(g, 64, 16, 512), _randn(g, 64, 2, 256), _randn(g, 64, 2, 256)
    got = qff.gqa_prefill_paged(small, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=1836, out_dtype=DT[out])
    pos = torch.arange(1836, 1900, dtype=torch.int32, device=DEV)
    assert_near(got, R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos), "", c.kv, fp16_operands=out == "f32")
    small.close()


def test_prefill_paged_against_64_bits(hip, ctx):
    """fp16 operands: 3e-4 of the row (four times it here), and the output's
    own rounding."""
    import qff
    c = Case([1000], 64, seed=31)
    g = torch.Generator(device=DEV).manual_seed(1)
    T, start = 130, 870
    qg, k, v = _randn(g, T, 16, 512), _randn(g, T, 2, 256), _randn(g, T, 2, 256)
    out = qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=start, out_dtype=torch.float32)
    pos = torch.arange(start, start + T, dtype=torch.int32, device=DEV)
    ref = R.attend(c.p, qg, c.kp, c.vp, c.table[0], pos)
    rel = ((out.double() - ref).norm(dim=-1) / ref.norm(dim=-1)).max()
    assert rel <= 1.2e-3, float(rel)


@pytest.mark.parametrize("T,kv", [(100, "bf16"), (129, "bf16"), (60, "bf16"), (100, "f16"), (9, "f16"), (8, "bf16"), (5, "f16"), (1, "bf16")])
def test_prefill_pages_outside_the_pool(hip, ctx, T, kv):
    """Rows that see a position without a page are NaN, rows before it are not."""
    import qff
    g = torch.Generator(device=DEV).manual_seed(2)
    start = 170 - T
    p = _params(g)
    qg, k, v = _randn(g, T, 16, 512), _randn(g, T, 2, 256), _randn(g, T, 2, 256)
    for entry, first in ((8, 128), (2, 0)) if T > 9 else ((2, 0),):    # positions 128 .. 143, or cached ones
        kp, vp = _randn(g, 13, 16, 2, 256, dtype=DT[kv]), _randn(g, 13, 16, 2, 256, dtype=DT[kv])
        kp[0], vp[0] = float("nan"), float("nan")     # nobody's
        table = torch.arange(1, 12, dtype=torch.int32, device=DEV)
        table[entry] = 13
        kb, vb = kp.clone(), vp.clone()
        out = qff.gqa_prefill_paged(ctx, p, qg, k, v, kp, vp, table, start_pos=start)
        nan = torch.isnan(out).all(dim=2).all(dim=1)
        assert torch.equal(nan, torch.arange(start, start + T, device=DEV) >= first)
        assert not torch.isnan(out[~nan]).any()
        for q in range(start, start + T):
            if q // 16 != entry:
                kb[1 + q // 16, q % 16], vb[1 + q // 16, q % 16] = kp[1 + q // 16, q % 16], vp[1 + q // 16, q % 16]
        assert same_bits(kb, kp) and same_bits(vb, vp)
        assert start > 160 or torch.equal(vp[11, 0], v[160 - start].to(DT[kv]))


def test_prefill_captured(hip, ctx):
    import qff
    c = Case([1000], 64, seed=41)
    g = torch.Generator(device=DEV).manual_seed(1)
    qg, k, v = _randn(g, 64, 16, 512), _randn(g, 64, 2, 256), _randn(g, 64, 2, 256)
    out = torch.empty(64, 16, 256, device=DEV)
    call = lambda o: qff.gqa_prefill_paged(ctx, c.p, qg, k, v, c.kp, c.vp, c.table[0], start_pos=900, out=o)  # noqa: E731
    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for _ in range(3):
        qg.normal_()
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(call(torch.empty_like(out)), got)


# ------------------------------------------------------------------ refusals

def test_refusals(hip, ctx):
    """What the library refuses on the host, with its status; nothing runs."""
    import ctypes

    import qff
    c = Case([100, 50], 64, seed=1)
    call = lambda **kw: qff.gqa_decode_paged(ctx, **{**dict(zip(  # noqa: E731
        ("params", "q_gate", "k_new", "v_new", "k_pages", "v_pages", "table", "positions"), c.args())), **kw})
    before = c.before()

    def refused(status, **kw):
        with pytest.raises(qff.QffError) as e:
            call(**kw)
        assert e.value.status == status

    refused(-2, k_pages=c.kp[:, :48].contiguous(), v_pages=c.vp[:, :48].contiguous())
    refused(-2, k_pages=c.kp[:, :8].contiguous(), v_pages=c.vp[:, :8].contiguous())
    refused(-4, table=torch.zeros(2, 65, dtype=torch.int32, device=DEV))    # 65 x 64 > 4096
    refused(-1, eps=-1.0)
    refused(-1, scale=float("inf"))
    refused(-1, table=torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    off = torch.empty(2 * 16 * 512 + 4, device=DEV)[1:-3].view(2, 16, 512)   # 4 bytes past a 16-byte boundary
    refused(-1, q_gate=off, k_new=c.k, v_new=c.v)
    for kw in ({"table": c.table[:1]}, {"positions": c.pos[:1]}, {"table": c.table.cpu()}, {"k_pages": c.kp[:, :, :1]},
               {"k_pages": c.kp.transpose(0, 1)}, {"out": torch.empty(1, 16, 256, device=DEV)},
               {"params": {k: w[:128] for k, w in c.p.items()}}):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in ({"table": c.table.long()}, {"positions": c.pos.long()}, {"k_pages": c.kp.float(), "v_pages": c.vp.float()},
               {"k_new": c.k.double()}, {"v_pages": c.vp.half()}):
        with pytest.raises(TypeError):
            call(**kw)
    with pytest.raises(qff.QffError) as e:   # larger than the context's batch
        n = 81
        qff.gqa_decode_paged(ctx, c.p, c.qg[:1].repeat(n, 1, 1), c.k[:1].repeat(n, 1, 1), c.v[:1].repeat(n, 1, 1), c.kp, c.vp,
                             c.table[:1].repeat(n, 1), c.pos[:1].repeat(n))
    assert e.value.status == -4
    one = dict(params=c.p, q_gate=c.qg, k=c.k, v=c.v, k_pages=c.kp, v_pages=c.vp, table=c.table[0])
    for kw, status in (({"start_pos": 127}, -1), ({"start_pos": -1}, -1),
                       ({"table": torch.zeros(64, dtype=torch.int32, device=DEV), "start_pos": 4095}, -1)):
        with pytest.raises(qff.QffError) as e:
            qff.gqa_prefill_paged(ctx, **{**one, **kw})
        assert e.value.status == status
    assert same_bits(before[0], c.kp)
    assert ctypes.sizeof(ctypes.c_void_p) == 8


# --------------------------------------------------------------------- copies

@pytest.mark.parametrize("shape,dtype", [((40, 16, 2, 256), torch.bfloat16), ((40, 3, 7, 8), torch.float32),
                                         ((40, 16), torch.uint8), ((40, 5, 1024, 1000), torch.float16)])
@pytest.mark.parametrize("pools", [1, 3, 33])
def test_pages_copy(hip, ctx, shape, dtype, pools):
    """Pages of 16 bytes to 10 MB (whole and partial 16 KB pieces), pools past
    one launch's; a source used more than once; everything else as it was."""
    import qff
    if pools == 33 and shape[1] == 5:
        shape = (40, 5, 64, 1000)
    g = torch.Generator(device=DEV).manual_seed(pools)
    ps = [(torch.rand(shape, device=DEV, generator=g) * 200).to(dtype) for _ in range(pools)]
    src, dst = [3, 3, 39, 7, 3], [0, 5, 6, 38, 12]
    want = [p.clone() for p in ps]
    for w in want:
        for a, b in zip(src, dst):
            w[b] = w[a]
    qff.pages_copy(ctx, ps, src, dst)
    for p, w in zip(ps, want):
        assert torch.equal(p, w)


@pytest.mark.parametrize("n", [0, 1, 447, 448, 449, 1500])
def test_pages_copy_many_pairs(hip, ctx, n):
    """Pairs past one launch's, and none."""
    import qff
    rng = np.random.default_rng(n)
    order = rng.permutation(3200).astype(np.int32)
    src, dst = torch.from_numpy(order[:n].copy()), torch.from_numpy(order[n:2 * n].copy())
    pool = torch.randn(3200, 4, 64, device=DEV)
    want = pool.clone()
    want[dst.long().to(DEV)] = pool[src.long().to(DEV)]
    qff.pages_copy(ctx, [pool], src, dst)
    assert torch.equal(pool, want)


def test_pages_copy_captured_and_refused(hip, ctx):
    import qff
    pool = torch.randn(10, 64, device=DEV)
    qff.pages_copy(ctx, [pool], [0], [1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    src, dst = torch.tensor([2, 3], dtype=torch.int32), torch.tensor([4, 5], dtype=torch.int32)
    with torch.cuda.graph(graph):
        qff.pages_copy(ctx, [pool], src, dst)
    src[:], dst[:] = 9, 8      # the captured pairs stay what they were
    for _ in range(3):
        pool.normal_()
        want = pool.clone()
        want[4], want[5] = pool[2], pool[3]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want)
    want = pool.clone()
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0]), ([10], [0]), ([0], [10]), ([-1], [0]), ([0], [-1])):
        with pytest.raises(qff.QffError) as e:
            qff.pages_copy(ctx, [pool], src, dst)
        assert e.value.status == -1
    with pytest.raises(qff.QffError) as e:
        qff.pages_copy(ctx, [pool[:, :3].contiguous()], [0], [1])    # 12 bytes a page
    assert e.value.status == -2
    with pytest.raises(ValueError):
        qff.pages_copy(ctx, [pool, pool[:5]], [0], [1])
    with pytest.raises(ValueError):
        qff.pages_copy(ctx, [], [0], [1])
    with pytest.raises(ValueError):
        qff.pages_copy(ctx, [pool], [0, 1], [2])
    with pytest.raises(TypeError):
        qff.pages_copy(ctx, [pool], torch.tensor([0]), torch.tensor([1]))
    torch.cuda.synchronize()
    assert torch.equal(pool, want)
    qff.pages_copy(ctx, [pool], [0], [1])   # (a refused call leaves no mark)
    want[1] = want[0]
    assert torch.equal(pool, want)
