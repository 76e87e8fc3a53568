"""What the planted rows of tests/paged_peaks.py can show, on the CPU: the online
softmax is right on them, and a maximum raised without rescaling the sum or the
output, rescaling at the wrong place, or joining chunks as if their maxima were
equal is far outside the tolerances of the GPU tests that use them."""
import random

import pytest
import torch

import paged_peaks as P
import paged_ref as R

BAR = 5e-6 * P.MOST / P.LOG2E      # of the GPU tests' fp32 rows


def _rows(seed, n=600, rows=3):
    g = torch.Generator().manual_seed(seed)
    w = 1 + 0.1 * torch.randn(256, generator=g)
    q = R.rope_norm(torch.randn(rows, 16, 256, generator=g), w, torch.arange(n, n + rows))
    K = torch.randn(n, 2, 256, generator=g).bfloat16().double()
    V = torch.randn(n, 2, 256, generator=g).double()
    picked = set()
    for p, j, k in P.ladders(q, n, random.Random(seed)):
        K[p, j] = k.bfloat16().double()
        picked.add((p, j))
    assert len(picked) > 100
    for r in range(rows):
        for h in range(16):
            yield (K[:, h // 8] @ q[r, h]) / 16 * P.LOG2E, V[:, h // 8]


def _worst(rows, **kw):
    """Error of each row relative to its norm, the largest first."""
    err = []
    for s, v in rows:
        ref = torch.softmax(s / P.LOG2E, 0) @ v
        err.append(float((P.online(s, v, **kw) - ref).norm() / ref.norm()))
    return sorted(err, reverse=True)


@pytest.mark.parametrize("tile,chunk", [(16, 64), (16, 640), (32, 192), (64, 256), (64, 640)])
def test_planted_rows_show_a_wrong_rescale(tile, chunk):
    rows = list(_rows(tile + chunk))
    assert max(float(s.max()) for s, _ in rows) <= 1.1 * P.MOST      # (others' rows score by chance, a little)
    raised = sum(any(float(s[t:t + tile].max()) > float(s[c:t].max()) + 8 for c in range(0, len(s), chunk)
                     for t in range(c + tile, min(c + chunk, len(s)), tile)) for s, _ in rows)
    assert raised >= 12 or chunk == 64
    assert _worst(rows, tile=tile, chunk=chunk)[0] < 1e-12
    for mistake in ("sum", "output", "late", "join"):
        if mistake == "join" and chunk > len(rows[0][0]):
            continue
        worst = _worst(rows, tile=tile, chunk=chunk, mistake=mistake)
        assert worst[5] > 20 * BAR, (mistake, worst[:8])


def test_normal_rows_would_not():
    """Why they are planted: with normal K no maximum is raised behind the first tile."""
    g = torch.Generator().manual_seed(1)
    s = torch.randn(200, 2048, generator=g).double() * P.LOG2E
    assert not (s[:, 64:].amax(1) > s[:, :64].amax(1) + 8).any()
