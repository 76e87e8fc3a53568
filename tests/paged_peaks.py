"""Inputs whose softmax has to be rescaled on the way, for the paged calls. With
normal K and normed q a row's first positions already hold about its maximum;
here chosen K rows lift a q row's score step by step, by 7.9, 8.1 or 40 in base
2 (the kernels raise a running maximum where it is passed by more than 8)."""
import torch

import paged_ref as R

STEPS = (7.9, 8.1, 7.9, 40.0)
LOG2E = 1.4426950408889634
MOST = 10 + 40 + 5 * 8.1    # the largest score, in base 2


def ladders(q, n, rng, each=6, part=0.5):
    """K rows for some of the positions 0 .. n - 1: for about `part` of the q
    rows (normed and rotated q [rows, 16, 256], 64 bits) `each` positions with
    rising scores. Yields (position, kv head, K row in 64 bits)."""
    for j in range(2):
        picks = [(r, h) for r in range(q.shape[0]) for h in range(8 * j, 8 * j + 8) if rng.random() < part]
        free = list(range(n))
        rng.shuffle(free)
        for r, h in picks:
            at, free = sorted(free[:each]), free[each:]
            t, far = rng.uniform(2, 10), False
            for p in at:
                yield p, j, q[r, h] * (t / LOG2E * 16 / q[r, h].square().sum())
                step = rng.choice(STEPS[:3] if far else STEPS)
                far |= step == 40.0
                t += step


def plant(case, members, lo, hi, rng, q=None, **kw):
    """Ladders at positions lo .. hi - 1 of the first member's table row, for the q
    rows of all members (or those given)."""
    if hi <= lo:
        return
    if q is None:
        q = torch.cat([R.rope_norm(case.qg[b:b + 1, :, :256], case.p["q_norm_w"], case.pos[b:b + 1]) for b in members])
    rows = list(ladders(q, hi - lo, rng, **kw))
    if not rows:
        return
    pos = torch.tensor([lo + p for p, _, _ in rows], device=q.device)
    kv = torch.tensor([j for _, j, _ in rows], device=q.device)
    at = case.table[members[0]].long()[pos // case.page]
    case.kp[at, pos % case.page, kv] = torch.stack([k for _, _, k in rows]).to(case.kp.dtype)


def online(s, v, tile, chunk, lazy=8.0, mistake=None):
    """Softmax over scores s [n] (base 2) times v [n, d], as the kernels take it:
    tile after tile of a chunk with a running maximum that is raised where it is
    passed by more than `lazy`, the chunks joined by their maxima. `mistake`: what is
    left out or done in the wrong order."""
    parts = []
    for c in range(0, len(s), chunk):
        m, d, o = -torch.inf, torch.zeros((), dtype=s.dtype), torch.zeros(v.shape[1], dtype=s.dtype)
        for t in range(c, min(c + chunk, len(s)), tile):
            x, y = s[t:min(t + tile, c + chunk)], v[t:min(t + tile, c + chunk)]
            alpha = 1.0
            if float(x.max()) > m + lazy:
                alpha, m = 2.0 ** (m - float(x.max())), float(x.max())
            e = torch.exp2(x - m)
            if mistake == "late":      # the new products scaled along with the old
                d, o = (d + e.sum()) * alpha if t > c else e.sum(), (o + e @ y) * alpha if t > c else e @ y
                continue
            d = d * (1.0 if mistake == "sum" and t > c else alpha) + e.sum()
            o = o * (1.0 if mistake == "output" and t > c else alpha) + e @ y
        parts.append((m, d, o))
    M = max(m for m, _, _ in parts)
    w = [1.0 if mistake == "join" else 2.0 ** (m - M) for m, _, _ in parts]
    return sum(f * o for f, (_, _, o) in zip(w, parts)) / sum(f * d for f, (_, d, _) in zip(w, parts))
