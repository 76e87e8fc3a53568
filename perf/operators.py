"""Timed cases of the paged KV cache and the attention that reads it: what a
program that serves many sequences of the hybrid stack from one pool of pages
calls, each through the public entry points of `qff` on one GPU.

  decode    one decode step of a full-attention layer, every sequence's cache
            rows found through its row of a page table
  shared    the same step where groups of sequences (samples of one prompt,
            requests under one system prompt) hold the same first pages
  prefill   a prompt slice of one sequence, attended over its pages and
            appended to them
  copy      pages of one or several pools copied: a fork's last page, a
            compaction, a fork of recurrent states

With `own` false, `run` computes them in elementary torch operations in 32
bits (RoPE angles in 64); with `own` true it calls the framework. `exact`
restates the definitions in float64, sequence by sequence.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
THETA, SCALE, EPS = 1e7, 1.0 / 16, 1e-6
POSITION = 1024          # values of one position in one pool's page: 2 kv heads x 256, K and V pools each half of it
MOST_CTX, MOST_BATCH = 65536, 32


def listed():
    return [
        # a single user's short chat: the smallest step, bound by latency (fp32 activations, as the stack keeps them)
        {"name": "decode_b1_1k", "op": "decode", "batch": 1, "ctx": 1000, "page": 16, "io": "f32", "kv": "bf16"},
        # an ordinary decode batch of ragged lengths
        {"name": "decode_b8_8k", "op": "decode", "batch": 8, "ctx": 8192, "page": 64, "io": "bf16", "kv": "bf16"},
        # a full decode batch of long sequences, the reference's fp16 cache
        {"name": "decode_b32_32k", "op": "decode", "batch": 32, "ctx": 32768, "page": 64, "io": "f32", "kv": "f16"},
        # eight samples of one 4K prompt, a few hundred tokens into their answers
        {"name": "shared_b8_4k", "op": "shared", "batch": 8, "groups": 1, "prefix": 4096, "suffix": 500, "page": 64,
         "io": "bf16", "kv": "bf16"},
        # requests under three system prompts of different lengths, small pages
        {"name": "shared_b23_3x5k", "op": "shared", "batch": 23, "groups": 3, "prefix": 5000, "suffix": 700, "page": 16,
         "io": "f32", "kv": "bf16"},
        # a full batch over one long document
        {"name": "shared_b32_32k", "op": "shared", "batch": 32, "groups": 1, "prefix": 32768, "suffix": 1000, "page": 64,
         "io": "bf16", "kv": "f16"},
        # a short chat turn behind a short history (fp32 activations)
        {"name": "prefill_t33_900", "op": "prefill", "T": 33, "start": 900, "page": 16, "io": "f32", "kv": "bf16"},
        # a chat turn behind a long history (ragged: neither is a multiple of a page), fp16 cache
        {"name": "prefill_t500_12k", "op": "prefill", "T": 500, "start": 12011, "page": 64, "io": "bf16", "kv": "f16"},
        # a long prompt into empty pages: the largest call
        {"name": "prefill_t8192", "op": "prefill", "T": 8192, "start": 0, "page": 64, "io": "bf16", "kv": "bf16"},
        # one sequence forked: its last page in the K and V pools of ten layers
        {"name": "copy_fork_page", "op": "copy", "pools": 20, "pages": 300, "pairs": 1, "kib": 64, "dtype": "bf16"},
        # a compaction after many sequences ended: an odd number of small pages moved in every pool
        {"name": "copy_compact", "op": "copy", "pools": 20, "pages": 5000, "pairs": 1777, "kib": 16, "dtype": "f16"},
        # seven children forked from one sequence: its fp32 DeltaNet state in thirty layers
        {"name": "copy_fork_state", "op": "copy", "pools": 30, "pages": 8, "pairs": 7, "kib": 2048, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "shared", "prefill", "copy"])
    page, io, kv = rng.choice([16, 32, 64, 128, 256]), rng.choice(["f32", "bf16"]), rng.choice(["bf16", "f16"])
    if op == "decode":
        batch = _log(rng, 1, MOST_BATCH)
        return {"op": op, "batch": batch, "ctx": _log(rng, 100, min(MOST_CTX, 32 * 32768 // batch)), "page": page, "io": io, "kv": kv}
    if op == "shared":
        batch = rng.randint(2, MOST_BATCH)
        groups = _log(rng, 1, max(1, batch // 2))
        return {"op": op, "batch": batch, "groups": groups, "prefix": _log(rng, 256, 32768),
                "suffix": _log(rng, 20, 1000), "page": page, "io": io, "kv": kv}
    if op == "prefill":
        T = _log(rng, 2, 8000)
        start = rng.choice([0, _log(rng, 1, min(MOST_CTX - T, 8192 * 4096 // T - T // 2 + 1))])
        return {"op": op, "T": T, "start": start, "page": page, "io": io, "kv": kv}
    pairs, kib = _log(rng, 1, 1500), rng.choice([16, 32, 64, 128])
    pools = _log(rng, 1, max(1, min(20, 500_000 // (pairs * kib))))
    return {"op": op, "pools": pools, "pages": 2 * pairs + rng.randint(1, 400), "pairs": pairs, "kib": kib,
            "dtype": rng.choice(["f32", "bf16", "f16"])}


# ------------------------------------------------------------------- inputs

_ctx = None


def _context():
    """The one context a program creates (default limits) and keeps."""
    global _ctx
    if _ctx is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-fieldfare_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import qff
        _ctx = qff.Context()
    return _ctx


def _randn(gen, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(mean, std, generator=gen)


def _spread(most, n):
    """n lengths over 1 .. most, the longest among them: the same total for every seed."""
    return [max(1, most * (i + 1) // n) for i in range(n)]


def _groups(case):
    """(first sequence, sequences, shared positions) of each group: whole pages, the last group's prefix the longest."""
    B, G, page = case["batch"], case["groups"], case["page"]
    at = [B * g // G for g in range(G + 1)]
    return [(at[g], at[g + 1] - at[g], max(page, case["prefix"] * (g + 1) // G // page * page)) for g in range(G)]


def _lengths(case):
    """Attended positions of each sequence, the new token among them, before the seed orders them: [B]."""
    if case["op"] == "decode":
        return _spread(case["ctx"], case["batch"])
    n = _spread(case["suffix"], case["batch"])
    return [S + n[b] for first, m, S in _groups(case) for b in range(first, first + m)]


def _inputs(case, seed):
    """What prepare() and exact() both start from."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.default_rng(seed)
    if case["op"] == "copy":
        shape = (case["pages"], case["kib"] * 1024 // SIZE[case["dtype"]])
        order = r.permutation(case["pages"])
        n = case["pairs"]
        # a fork reads one page many times, a compaction many pages once
        src = order[n:n + 1].repeat(n) if case["pages"] < 2 * n else order[n:2 * n]
        return {"pools": [_randn(g, shape, DT[case["dtype"]]) for _ in range(case["pools"])],
                "src": torch.from_numpy(src.astype(np.int32)), "dst": torch.from_numpy(order[:n].astype(np.int32))}
    page, io, kv = case["page"], DT[case["io"]], DT[case["kv"]]
    if case["op"] == "prefill":
        n, lengths = case["T"], [case["start"] + case["T"]]
        group = None
    else:
        n, lengths = case["batch"], _lengths(case)
        if case["op"] == "decode":
            lengths = [lengths[i] for i in r.permutation(n)]
            group = None
        else:
            group = _groups(case)
    cols = -(-max(lengths) // page)
    need = [-(-L // page) for L in lengths]
    own_pages = list(need)
    if group:
        for first, m, S in group:
            for b in range(first + 1, first + m):
                own_pages[b] -= S // page
    total = sum(own_pages)
    num = total + total // 16 + 1   # a few pages free, as a pool in use has
    order = r.permutation(num)[:total].astype(np.int32)
    table = np.full((len(lengths), cols), -1, np.int32)
    at = 0
    leader = {b: (first, S // page) for first, m, S in group or [] for b in range(first + 1, first + m)}
    for b, k in enumerate(need):
        lead, have = leader.get(b, (b, 0))
        table[b, :have] = table[lead, :have]
        table[b, have:k] = order[at:at + k - have]
        at += k - have
    s = {"p": {name: _randn(g, 256, std=0.1, mean=1.0).bfloat16().float() for name in ("q_norm_w", "k_norm_w")},
         "qg": _randn(g, (n, 16, 512), io), "k": _randn(g, (n, 2, 256), io), "v": _randn(g, (n, 2, 256), io),
         "kp": _randn(g, (num, page, 2, 256), kv), "vp": _randn(g, (num, page, 2, 256), kv),
         "table": torch.from_numpy(table).to(DEV)}
    if case["op"] != "prefill":
        s["pos"] = torch.tensor([L - 1 for L in lengths], dtype=torch.int32, device=DEV)
    if group:
        s["group"] = torch.tensor([i for i, (_, m, _) in enumerate(group) for _ in range(m)], dtype=torch.int32, device=DEV)
        s["shared"] = torch.tensor([S for _, m, S in group for _ in range(m)], dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if case["op"] == "copy":
        s["src_dev"], s["dst_dev"] = s["src"].long().to(DEV), s["dst"].long().to(DEV)
    else:
        # a prompt slice's rows are kept in 16 bits, a decode step's in its activations' type
        s["out"] = torch.empty(s["qg"].shape[0], 16, 256, dtype=torch.bfloat16 if case["op"] == "prefill" else s["qg"].dtype, device=DEV)
    return s


# ---------------------------------------------------------------------- run

def run(s):
    if not own:
        return _plain(s)
    op, ctx = s["case"]["op"], _context()
    import qff
    if op == "copy":
        qff.pages_copy(ctx, s["pools"], s["src"], s["dst"])
        return s["pools"]
    if op == "decode":
        qff.gqa_decode_paged(ctx, s["p"], s["qg"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["pos"], out=s["out"])
    elif op == "shared":
        qff.gqa_decode_shared(ctx, s["p"], s["qg"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["pos"], s["group"],
                              s["shared"], out=s["out"])
    else:
        qff.gqa_prefill_paged(ctx, s["p"], s["qg"], s["k"], s["v"], s["kp"], s["vp"], s["table"][0],
                              start_pos=s["case"]["start"], out=s["out"])
    return {"out": s["out"], "k_pages": s["kp"], "v_pages": s["vp"]}


def _frequencies():
    """1 / theta^(2i / 64), i < 32, as the model holds them: a 32-bit power and a 32-bit quotient."""
    e = np.arange(32, dtype=np.float32) * np.float32(2) / np.float32(64)
    return torch.from_numpy(np.float32(1) / np.power(np.float64(np.float32(THETA)), e.astype(np.float64)).astype(np.float32)).to(DEV)


def _norm_rope(x, w, pos):
    """Head RMS norm and rotation of the first 64 dims (pairs i, i + 32) of x [n, heads, 256]; the angle is the
    32-bit product of position and frequency, its sine and cosine taken in 64 bits."""
    x = x.float()
    x = x * (x.square().mean(2, keepdim=True) + EPS).rsqrt() * w
    ang = (pos.float()[:, None] * _frequencies()[None, :]).double()
    c, s = torch.cos(ang).float()[:, None, :], torch.sin(ang).float()[:, None, :]
    lo, hi = x[:, :, :32], x[:, :, 32:64]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[:, :, 64:]], 2)


def _append(pages, table_row, pos, rows):
    """rows [n, 2, 256] into the places of positions pos [n]; table_row [n, cols]."""
    page = pages.shape[1]
    at = table_row.gather(1, (pos // page)[:, None].long())[:, 0].long()
    pages[at, (pos % page).long()] = rows.to(pages.dtype)


def _softmax_times(scores, mask, values):
    scores = scores.masked_fill_(mask, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.matmul(e, values) / e.sum(-1, keepdim=True)


def _plain(s):
    if s["case"]["op"] == "copy":
        for pool in s["pools"]:
            pool[s["dst_dev"]] = pool[s["src_dev"]]
        return s["pools"]
    qg, p, table, page = s["qg"], s["p"], s["table"], s["case"]["page"]
    n = qg.shape[0]
    if s["case"]["op"] == "prefill":
        pos = torch.arange(s["case"]["start"], s["case"]["start"] + n, dtype=torch.int32, device=DEV)
        rows = table.expand(n, -1)
    else:
        pos, rows = s["pos"], table
    q = _norm_rope(qg[:, :, :256], p["q_norm_w"], pos)
    _append(s["kp"], rows, pos, _norm_rope(s["k"], p["k_norm_w"], pos))
    _append(s["vp"], rows, pos, s["v"])
    # every table row's positions side by side: [sequences, 2, positions, 256]
    at = table.clamp(min=0).long()
    K = s["kp"][at].flatten(1, 2).permute(0, 2, 1, 3).float()
    V = s["vp"][at].flatten(1, 2).permute(0, 2, 1, 3).float()
    hidden = torch.arange(K.shape[2], device=DEV)[None, :] > pos[:, None]
    if s["case"]["op"] == "prefill":
        q = q.view(n, 2, 8, 256).permute(1, 2, 0, 3).reshape(1, 2, 8 * n, 256)
        hidden = hidden.repeat(8, 1)[None, None]
    else:
        q = q.view(n, 2, 8, 256)
        hidden = hidden[:, None, None]
    o = _softmax_times(torch.matmul(q, K.transpose(2, 3)) * SCALE, hidden, V)
    if s["case"]["op"] == "prefill":
        o = o.view(2, 8, n, 256).permute(2, 0, 1, 3)
    o = o.reshape(n, 16, 256) * torch.sigmoid(qg[:, :, 256:].float())
    s["out"].copy_(o)
    return {"out": s["out"], "k_pages": s["kp"], "v_pages": s["vp"]}


# --------------------------------------------------------------------- work

def work(case):
    """What a step cannot do without: each shared prefix, each other cached position and every activation once, two
    products of 256 dims for each of 16 heads and attended position."""
    if case["op"] == "copy":
        n = case["pairs"] if case["pages"] >= 2 * case["pairs"] else 1   # a forked page is read once
        return {"bytes": case["pools"] * (n + case["pairs"]) * case["kib"] * 1024, "flops": 0}
    io, row = SIZE[case["io"]], POSITION * SIZE[case["kv"]]
    if case["op"] == "prefill":
        n, T, s = case["T"], case["T"], case["start"]
        read, seen = s, T * s + T * (T + 1) // 2
    else:
        n, L = case["batch"], _lengths(case)
        read, seen = sum(L) - n, sum(L)
        if case["op"] == "shared":
            read -= sum((m - 1) * S for _, m, S in _groups(case))
    to = 2 if case["op"] == "prefill" else io
    return {"bytes": n * ((16 * 512 + 2 * 512) * io + 16 * 256 * to) + row * (read + n), "flops": 4 * 256 * 16 * seen}


# -------------------------------------------------- the same in 64-bit torch

def _rotated64(x, w, pos):
    """As the definition of _norm_rope, one row at a time's formula in 64 bits: x [n, heads, 256] double."""
    x = x / torch.sqrt((x * x).sum(2, keepdim=True) / 256 + EPS) * w.double()
    f = [float(np.float32(1) / np.float32(float(np.float32(THETA)) ** (2 * i / 64))) for i in range(32)]
    f = torch.tensor(f, dtype=torch.float32, device=DEV)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), (pos.float()[:, None] * f).double())[:, None, :]
    z = torch.complex(x[..., :32].contiguous(), x[..., 32:64].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[..., 64:]], -1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "copy":
        if case["pairs"] * case["pools"] > 40000:
            return None
        new = [pool.clone() for pool in s["pools"]]
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for pool, to in zip(s["pools"], new):
                to[b].copy_(pool[a])
        return new
    kp, vp, page = s["kp"].double(), s["vp"].double(), case["page"]
    qg, k, v = s["qg"].double(), s["k"].double(), s["v"].double()
    n = qg.shape[0]
    first = case["start"] if case["op"] == "prefill" else None
    pos = torch.arange(first, first + n, device=DEV) if first is not None else s["pos"].long()
    q, k = _rotated64(qg[:, :, :256], s["p"]["q_norm_w"], pos), _rotated64(k, s["p"]["k_norm_w"], pos)
    table, where = s["table"].tolist(), pos.tolist()
    # the attention reads the rows as the cache holds them, rounded to its type
    kc, vc = kp.clone(), vp.clone()
    for i, t in enumerate(where):
        at = table[0 if first is not None else i][t // page]
        kp[at, t % page], vp[at, t % page] = k[i], v[i]
        kc[at, t % page], vc[at, t % page] = k[i].to(s["kp"].dtype).double(), v[i].to(s["vp"].dtype).double()
    out = torch.empty(n, 16, 256, dtype=torch.float64, device=DEV)
    step = 128 if first is not None else 1
    for i in range(0, n, step):
        last = where[min(n, i + step) - 1]
        at = torch.tensor(table[0 if first is not None else i][:last // page + 1], device=DEV)
        seen = torch.arange(last + 1, device=DEV)[None, :] <= pos[i:i + step, None]
        for h in range(2):
            K, V = (c[at, :, h].reshape(-1, 256)[:last + 1] for c in (kc, vc))
            Q = q[i:i + step, 8 * h:8 * h + 8]
            e = (Q.reshape(-1, 256) @ K.t().contiguous() * SCALE).view(Q.shape[0], 8, -1)
            e = torch.softmax(e.masked_fill(~seen[:, None, :], -math.inf), -1)
            out[i:i + step, 8 * h:8 * h + 8] = (e.view(-1, last + 1) @ V).view(Q.shape[0], 8, 256)
    return {"out": out / (1 + torch.exp(-qg[:, :, 256:])), "k_pages": kp, "v_pages": vp}
