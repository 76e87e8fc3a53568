"""Positions past 2^25 of one sequence on pages: 34 million of them, whose pages
repeat four (a cached page may be named any number of times), so that a small
pool holds them and the 64-bit reference is a sum over four pages' rows with
their counts.

Tolerances as in tests/test_gpu_gqa_paged.py (fp32 outputs: 5e-6 of a row for the
decode's kernels, 1.2e-3 for the fp16 operands of long slices) times 4 for the
decode's: a row's sums have 2^16 terms a chunk, whose fp32 rounding, 2^-24 / sqrt(3)
of the running sum each, adds up to 2^8 2^-25 = 8e-6 if it is random."""
import pytest
import torch

import paged_ref as R
from gpu_util import DEV

pytestmark = pytest.mark.gpu

PAGE, LAST = 4096, 2 ** 25 + 300_000
N = -(-LAST // PAGE)


@pytest.fixture(scope="module")
def far():
    import qff
    g = torch.Generator(device=DEV).manual_seed(1)
    c = qff.Context(max_batch=1, max_ctx=N * PAGE, max_prefill_tokens=128)   # 70 GB of workspace
    kp, vp = (torch.randn(6, PAGE, 2, 256, device=DEV, generator=g).bfloat16() for _ in range(2))
    table = torch.randint(0, 4, (N,), device=DEV, generator=g, dtype=torch.int32)
    table[-2:] = torch.tensor([4, 5], device=DEV)     # the slice's own
    p = {k: 1 + 0.1 * torch.randn(256, device=DEV, generator=g) for k in ("q_norm_w", "k_norm_w")}
    yield c, kp, vp, table, p, g
    c.close()


def _attend(p, qg, kp, vp, table, pos):
    """R.attend, with each of the repeated pages' rows once and its count's
    logarithm added to its score."""
    q = R.rope_norm(qg[:, :, :256], p["q_norm_w"], pos)
    count = torch.bincount(table[:-2].long(), minlength=4).double().log()
    start = (N - 2) * PAGE
    K, V = kp.flatten(0, 1).double(), vp.flatten(0, 1).double()
    more = torch.cat([count.repeat_interleave(PAGE), torch.zeros(2 * PAGE, device=DEV, dtype=torch.float64)])
    where = torch.cat([torch.zeros(4 * PAGE, device=DEV, dtype=torch.int64), start + torch.arange(2 * PAGE, device=DEV)])
    out = torch.empty(qg.shape[0], 16, 256, dtype=torch.float64, device=DEV)
    for h in range(16):
        s = (q[:, h].contiguous() @ K[:, h // 8].t().contiguous()) / 16 + more
        s = s.masked_fill(where[None, :] > pos[:, None].long(), -torch.inf)
        out[:, h] = torch.softmax(s, 1) @ V[:, h // 8].contiguous()
    return out * torch.sigmoid(qg[:, :, 256:].double())


@pytest.mark.parametrize("T,bar", [(1, 2e-5), (40, 2e-5), (70, 1.2e-3)])
def test_prefill_behind_33_million_positions(hip, far, T, bar):
    import qff
    c, kp, vp, table, p, g = far
    qg, k, v = (torch.randn(T, *s, device=DEV, generator=g) for s in ((16, 512), (2, 256), (2, 256)))
    start = LAST - T
    out = qff.gqa_prefill_paged(c, p, qg, k, v, kp, vp, table, start_pos=start, out_dtype=torch.float32)
    pos = torch.arange(start, LAST, device=DEV, dtype=torch.int32)
    ref = _attend(p, qg, kp, vp, table, pos)
    rel = ((out.double() - ref).norm(dim=-1) / ref.norm(dim=-1)).max()
    assert rel <= bar, float(rel)


def test_decode_behind_33_million_positions(hip, far):
    import qff
    c, kp, vp, table, p, g = far
    qg, k, v = (torch.randn(1, *s, device=DEV, generator=g) for s in ((16, 512), (2, 256), (2, 256)))
    pos = torch.tensor([LAST - 1], device=DEV, dtype=torch.int32)
    out = qff.gqa_decode_paged(c, p, qg, k, v, kp, vp, table[None], pos, out_dtype=torch.float32)
    ref = _attend(p, qg, kp, vp, table, pos)
    rel = ((out.double() - ref).norm(dim=-1) / ref.norm(dim=-1)).max()
    assert rel <= 2e-5, float(rel)
