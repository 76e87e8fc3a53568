"""Timed cases of what follows a layer's attention on the way to a token: the
expert block on affine-Q4 weights and the choice of the next token, each
through the public entry points of `qff` on one GPU.

  norm      RMSNorm of every token, with the shared expert's coefficient
            sigmoid(<normed token, Q8 row>) in the same pass
  gate_up   every token through its experts' gate and up projections (and the
            shared expert's): silu(x Wg^T) * (x Wu^T)
  down      the experts' down projections, weighted and summed for each
            token, on top of a residual
  sample    the next token of each sequence from its logits: temperature,
            top-k, top-p, min-p, with the random numbers as inputs

With `own` false, `run` computes them in elementary torch operations in 32
bits (sampling in 64: its results are whole numbers next to borders); with
`own` true it calls the framework. `exact` restates the definitions in
float64, expert by expert and row by row.
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
EPS = 1e-6
Q4_VALUE = 0.5 + 4 / 64      # bytes of a weight: a nibble and its share of a group's 16-bit scale and bias
MOST_TOKENS, MOST_VOCAB, MOST_BATCH = 8192, 262144, 32
UNIT = 2.0 ** 44             # a probability mass is held as a whole number of 2^-44 of the likeliest token's


def listed():
    moe = {"experts": 256, "top": 8, "hidden": 2048, "inter": 512, "shared": True, "sb": "bf16", "skew": 0.0, "pad": 0}
    return [
        # one token of a single user: the smallest call, fp32 activations as the stack keeps them
        {"name": "norm_t1", "op": "norm", "tokens": 1, "cols": 2048, "x": "f32", "y": "f32", "gate": True},
        # a long prompt's tokens ahead of the experts, to 16 bits
        {"name": "norm_t8192", "op": "norm", "tokens": 8192, "cols": 2048, "x": "f32", "y": "bf16", "gate": True},
        # a single user's decode step: nine experts' weights read once
        {"name": "gate_up_t1", "op": "gate_up", "tokens": 1, **moe, "x": "f32", "h": "f32"},
        # a full decode batch: most experts have one token or none
        {"name": "gate_up_t32", "op": "gate_up", "tokens": 32, **moe, "x": "f32", "h": "f32"},
        # a chat turn with unevenly used experts, its last tokens padding
        {"name": "gate_up_t500", "op": "gate_up", "tokens": 500, **moe, "skew": 1.0, "pad": 13, "x": "f32", "h": "f16"},
        # a long prompt
        {"name": "gate_up_t8192", "op": "gate_up", "tokens": 8192, **moe, "x": "bf16", "h": "f16"},
        # the decode steps' second half, on top of the fp32 residual stream
        {"name": "down_t1", "op": "down", "tokens": 1, **moe, "h": "f32", "y": "f32", "residual": True},
        {"name": "down_t32", "op": "down", "tokens": 32, **moe, "h": "f32", "y": "f32", "residual": True},
        # a chat turn on the fp32 residual stream (fp32 results whatever the size)
        {"name": "down_t500", "op": "down", "tokens": 500, **moe, "skew": 1.0, "pad": 13, "h": "f32", "y": "f32", "residual": True},
        # a long prompt kept in 16 bits: the largest call
        {"name": "down_t8192", "op": "down", "tokens": 8192, **moe, "h": "f16", "y": "bf16", "residual": True},
        # one user's next token with the usual settings
        {"name": "sample_b1", "op": "sample", "batch": 1, "vocab": 151936, "logits": "f32", "mode": "usual"},
        # a full batch whose requests each have settings of their own, greedy and unfiltered ones among them
        {"name": "sample_b32", "op": "sample", "batch": 32, "vocab": 151936, "logits": "f32", "mode": "mixed"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "gate_up", "gate_up", "down", "down", "sample"])
    if op == "norm":
        cols = 64 * _log(rng, 2, 64)
        return {"op": op, "tokens": _log(rng, 1, min(MOST_TOKENS, MOST_TOKENS * 2048 // cols)), "cols": cols,
                "x": rng.choice(["f32", "bf16"]), "y": rng.choice(["f32", "bf16"]), "gate": rng.random() < 0.5}
    if op == "sample":
        batch = _log(rng, 1, MOST_BATCH)
        return {"op": op, "batch": batch, "vocab": _log(rng, 500, min(MOST_VOCAB, 32 * 151936 // batch)),
                "logits": rng.choice(["f32", "bf16"]), "mode": rng.choice(["usual", "mixed"])}
    experts, top = rng.choice([8, 60, 64, 128, 256]), rng.choice([1, 2, 4, 6, 8])
    hidden, inter = 64 * _log(rng, 8, 64), 64 * _log(rng, 2, 32)
    while experts * hidden * inter > 256 * 2048 * 512:
        hidden, inter = max(512, hidden // 128 * 64), max(128, inter // 128 * 64)
        if hidden == 512 and inter == 128:
            break
    shared = rng.random() < 0.7
    most = MOST_TOKENS * 9 * 2048 * 512 // ((top + shared) * hidden * inter)
    tokens = _log(rng, 1, min(MOST_TOKENS, most))
    case = {"op": op, "tokens": tokens, "experts": experts, "top": top, "hidden": hidden, "inter": inter, "shared": shared,
            "sb": rng.choice(["bf16", "f16"]), "skew": rng.choice([0.0, 1.0]), "pad": rng.choice([0, tokens // 7])}
    if op == "gate_up":
        return {**case, "x": rng.choice(["f32", "bf16"]), "h": rng.choice(["f32", "bf16", "f16"])}
    return {**case, "h": rng.choice(["f32", "bf16", "f16"]), "y": rng.choice(["f32", "bf16"]), "residual": rng.random() < 0.7}


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


def _quantized(g, shape, cols, bits, dtype):
    """Affine-quantized matrices [*shape, cols] of groups of 64, values of about N(0, 1 / cols): words, scales, biases."""
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (*shape, cols * bits // 32), dtype=torch.int32, device=DEV, generator=g)
    top = 2 ** bits - 1
    s = torch.empty(*shape, cols // 64, device=DEV).uniform_(0.5, 1.5, generator=g).mul_(3.4 / top / math.sqrt(cols)).to(dtype)
    b = s.float().mul_(-top / 2).add_(_randn(g, s.shape, std=0.3 / math.sqrt(cols))).to(dtype)
    return w, s, b


def _popularity(case):
    """Each expert's logit ahead of a token's own: even, or spread as a router's may be without balancing."""
    n = case["experts"]
    return [case["skew"] * 2.0 * ((i * 0.6180339887) % 1.0 - 0.5) for i in range(n)]


def _used(case):
    """The experts that a call uses, as they are expected: an expert's chance to be among a token's is near
    1 - exp(-c w) for the c that makes the chances sum to top."""
    w = [math.exp(v) for v in _popularity(case)]
    n, top = case["tokens"] - case["pad"], min(case["top"], case["experts"])
    if top == case["experts"]:
        return top if n else 0
    lo, hi = 0.0, 1e6
    for _ in range(100):
        c = (lo + hi) / 2
        lo, hi = (c, hi) if sum(1 - math.exp(-c * v) for v in w) < top else (lo, c)
    return sum(1 - math.exp(-c * v * n) for v in w)


def _inputs(case, seed):
    """What prepare() and exact() both start from."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "norm":
        n, c = case["tokens"], case["cols"]
        # a residual stream: tokens of different size, a few large channels
        x = _randn(g, (n, c)) * torch.exp(_randn(g, (n, 1), std=0.5)) * torch.exp(_randn(g, (1, c), std=0.5))
        s = {"x": x.to(DT[case["x"]]), "w": _randn(g, c, std=0.1, mean=1.0).bfloat16().float()}
        if case["gate"]:
            s["gate"] = _quantized(g, (1,), c, 8, torch.bfloat16)
        return s
    if case["op"] == "sample":
        B, V = case["batch"], case["vocab"]
        logits = (_randn(g, (B, V)) * 2.0 + 6.0 * torch.rand(B, V, device=DEV, generator=g).pow(40)).to(DT[case["logits"]])
        s = {"logits": logits, "u": torch.rand(B, device=DEV, generator=g)}
        r = np.random.default_rng(seed)
        if case["mode"] == "usual":
            t, k, p, m = [0.8] * B, [50] * B, [0.95] * B, [0.0] * B
        else:
            # greedy, unfiltered, and each filter alone and with others
            t = [0.0 if i % 8 == 7 else float(r.uniform(0.5, 1.5)) for i in range(B)]
            k = [int(r.integers(1, 200)) if i % 8 in (1, 4, 6) else 0 for i in range(B)]
            p = [float(r.uniform(0.5, 0.99)) if i % 8 in (2, 4, 5, 6) else 1.0 for i in range(B)]
            m = [float(r.uniform(0.01, 0.2)) if i % 8 in (3, 5, 6) else 0.0 for i in range(B)]
        for name, v, dt in (("temperature", t, torch.float32), ("top_k", k, torch.int32), ("top_p", p, torch.float32),
                            ("min_p", m, torch.float32)):
            s[name] = torch.tensor(v, dtype=dt, device=DEV)
        return s
    n, E, D, I, sb = case["tokens"], case["experts"], case["hidden"], case["inter"], DT[case["sb"]]
    # Gumbel noise on the experts' popularity: a token's experts are drawn without repetition
    z = torch.tensor(_popularity(case), device=DEV) - torch.log(-torch.log(torch.rand(n, E, device=DEV, generator=g).clamp_(1e-20, 1 - 1e-7)))
    top = z.topk(min(case["top"], E), dim=1)
    idx = top.indices.to(torch.int32)
    if case["pad"]:
        idx[n - case["pad"]:] = -1
    slots = idx.shape[1] + case["shared"]
    s = {"indices": idx}
    if case["op"] == "gate_up":
        s["x"] = _randn(g, (n, D), DT[case["x"]])
        s["gate"], s["up"] = (_quantized(g, (E, I), D, 4, sb) for _ in range(2))
        if case["shared"]:
            s["shared_gate"], s["shared_up"] = (_quantized(g, (I,), D, 4, sb) for _ in range(2))
        return s
    a, b = _randn(g, (n, slots, I)), _randn(g, (n, slots, I))
    s["h"] = (a * torch.sigmoid(a) * b).to(DT[case["h"]])
    s["scores"] = torch.softmax(top.values, 1)
    s["down"] = _quantized(g, (E, D), I, 4, sb)
    if case["shared"]:
        s["shared_down"] = _quantized(g, (D,), I, 4, sb)
        s["coef"] = torch.sigmoid(_randn(g, n))
    if case["residual"]:
        s["residual"] = _randn(g, (n, D), DT[case["y"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    n = case.get("tokens")
    if case["op"] == "norm":
        s["out"] = torch.empty(n, case["cols"], dtype=DT[case["y"]], device=DEV)
        s["out_coef"] = torch.empty(n, device=DEV) if case["gate"] else None
    elif case["op"] == "gate_up":
        # (a padded token's rows are left as they were)
        s["out"] = torch.zeros(n, s["indices"].shape[1] + case["shared"], case["inter"], dtype=DT[case["h"]], device=DEV)
    elif case["op"] == "down":
        s["out"] = torch.empty(n, case["hidden"], dtype=DT[case["y"]], device=DEV)
    else:
        s["out"] = torch.empty(case["batch"], dtype=torch.int32, device=DEV)
        s["out_prob"] = torch.empty(case["batch"], device=DEV)
    return s


# ---------------------------------------------------------------------- run

def run(s):
    if not own:
        return {"norm": _plain_norm, "gate_up": _plain_gate_up, "down": _plain_down, "sample": _plain_sample}[s["case"]["op"]](s)
    op, ctx = s["case"]["op"], _context()
    import qff
    if op == "norm":
        qff.rms_norm(ctx, s["x"], s["w"], EPS, gate=s.get("gate"), out=s["out"], coef=s["out_coef"])
        return [s["out"], s["out_coef"]]
    if op == "sample":
        qff.sample(ctx, s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], out=s["out"], prob=s["out_prob"])
        return [s["out"], s["out_prob"]]
    if "experts" not in s:   # the handle of a layer's weights that a program makes once
        s["experts"] = qff.ExpertWeights(*(s.get(k) for k in ("gate", "up", "down", "shared_gate", "shared_up", "shared_down")))
    if op == "gate_up":
        return qff.moe_gate_up(ctx, s["experts"], s["x"], s["indices"], out=s["out"])
    return qff.moe_down(ctx, s["experts"], s["h"], s["indices"], s["scores"], coef=s.get("coef"), residual=s.get("residual"),
                        out=s["out"])


def _dequantized(w, s, b, bits):
    """[.., cols] float32 of words, scales and biases."""
    per = 32 // bits
    q = (w[..., None] >> (bits * torch.arange(per, dtype=torch.int32, device=DEV))) & (2 ** bits - 1)
    q = q.view(*w.shape[:-1], -1, 64).float()
    return (q * s.float()[..., None] + b.float()[..., None]).view(*w.shape[:-1], -1)


def _plain_norm(s):
    x = s["x"].float()
    y = x * (x.square().mean(1, keepdim=True) + EPS).rsqrt() * s["w"]
    s["out"].copy_(y)
    if s["out_coef"] is not None:
        s["out_coef"].copy_(torch.sigmoid((y * _dequantized(*s["gate"], 8)).sum(1)))
    return [s["out"], s["out_coef"]]


def _grouped(x, indices, weights):
    """Row p of x [pairs, cols] times the matrix of expert indices[p] (a pair without one: zeros): [pairs, rows], float32."""
    w, sc, bi = weights
    E, pairs = w.shape[0], x.shape[0]
    e = torch.where((indices >= 0) & (indices < E), indices, E).long()
    if pairs <= 2 * E // 3:   # few: each pair's own copy of its matrix
        at = e.clamp(max=E - 1)
        y = torch.matmul(_dequantized(w[at], sc[at], bi[at], 4), x[:, :, None])[:, :, 0]
        return y * (e < E)[:, None]
    # many: every expert's rows side by side, as many places as the fullest has
    counts = torch.bincount(e, minlength=E + 1)
    order = torch.argsort(e, stable=True)
    place = torch.arange(pairs, device=DEV) - (torch.cumsum(counts, 0) - counts)[e[order]]
    most = int(counts[:E].max())
    rows = torch.zeros(E + 1, max(most, int(counts[E]), 1), x.shape[1], device=DEV)
    rows[e[order], place] = x[order]
    rows = rows[:E, :max(most, 1)].transpose(1, 2).contiguous()
    y = torch.matmul(_dequantized(w, sc, bi, 4), rows)
    y = torch.cat([y, torch.zeros_like(y[:1])])
    out = torch.empty(pairs, w.shape[1], device=DEV)
    out[order] = y.transpose(1, 2)[e[order], place.clamp(max=max(most, 1) - 1)]
    return out


def _plain_gate_up(s):
    idx, x = s["indices"], s["x"].float()
    n, top = idx.shape
    pairs, flat = x.repeat_interleave(top, 0), idx.reshape(-1)
    g, u = _grouped(pairs, flat, s["gate"]), _grouped(pairs, flat, s["up"])
    h = (g * torch.sigmoid(g) * u).view(n, top, -1)
    has = ((idx >= 0) & (idx < s["gate"][0].shape[0]))[:, :, None]
    s["out"][:, :top] = torch.where(has, h.to(s["out"].dtype), s["out"][:, :top])
    if "shared_gate" in s:
        g = torch.matmul(x, _dequantized(*s["shared_gate"], 4).t())
        s["out"][:, top] = g * torch.sigmoid(g) * torch.matmul(x, _dequantized(*s["shared_up"], 4).t())
    return s["out"]


def _plain_down(s):
    idx, h = s["indices"], s["h"].float()
    n, top = idx.shape
    y = _grouped(h[:, :top].reshape(n * top, -1), idx.reshape(-1), s["down"]).view(n, top, -1)
    y = (y * s["scores"][:, :, None]).sum(1)
    if "shared_down" in s:
        y = y + torch.matmul(h[:, top], _dequantized(*s["shared_down"], 4).t()) * s["coef"][:, None]
    if "residual" in s:
        y = y + s["residual"].float()
    s["out"].copy_(y)
    return s["out"]


def _plain_sample(s):
    l = s["logits"].double()
    l = torch.where(l.isnan(), -math.inf, l)
    B, V = l.shape
    best = l.amax(1, keepdim=True)
    t, p, m = (s[k].double()[:, None] for k in ("temperature", "top_p", "min_p"))
    k = s["top_k"].long()[:, None]
    e = torch.exp(torch.where(l == best, 0.0, (l - best) / t))
    e = torch.where((l == -math.inf) | ~((t > 0) | (l == best)), 0.0, e)
    mass = torch.round(e * UNIT).long()
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    in_order = mass.gather(1, order)
    j = torch.arange(V, device=DEV)[None, :]
    keep = (j < torch.where(k > 0, k, V)) & ((e.gather(1, order) >= m) | ~(m > 0))
    head = torch.where(j < torch.where(k > 0, k, V), in_order, 0)
    keep &= ((torch.cumsum(head, 1) - head).double() < p * head.sum(1, keepdim=True).double()) | ~(p < 1)
    keep = (keep & (t > 0)) | (j == 0)
    kept = torch.zeros_like(mass).scatter_(1, order, torch.where(keep, in_order, 0))
    total = kept.sum(1, keepdim=True)
    aim = torch.floor(s["u"].double()[:, None].clamp(0, 1) * total.double()).long().minimum(total - 1).clamp(min=0)
    token = (torch.cumsum(kept, 1) <= aim).sum(1, keepdim=True)
    some = total > 0
    s["out"].copy_(torch.where(some, token, -1)[:, 0])
    s["out_prob"].copy_(torch.where(some, kept.gather(1, token.clamp(max=V - 1)).double() / total.double(), 0.0)[:, 0])
    return [s["out"], s["out_prob"]]


# --------------------------------------------------------------------- work

def work(case):
    """What a pass cannot do without: the weights of the experts that it uses, every activation and logit once, and the
    products (one of a token with each of its experts' rows)."""
    if case["op"] == "norm":
        n, c = case["tokens"], case["cols"]
        per = SIZE[case["x"]] + SIZE[case["y"]]
        return {"bytes": n * c * per + 4 * c + case["gate"] * (4 * n + c * (1 + 4 / 64)), "flops": n * c * (4 + 2 * case["gate"])}
    if case["op"] == "sample":
        # each logit read once and, to be weighed, exponentiated once
        return {"bytes": case["batch"] * (case["vocab"] * SIZE[case["logits"]] + 28), "flops": case["batch"] * case["vocab"]}
    n, D, I = case["tokens"], case["hidden"], case["inter"]
    top = min(case["top"], case["experts"])
    pairs = (n - case["pad"]) * top + n * case["shared"]
    matrices = 2 if case["op"] == "gate_up" else 1
    weights = matrices * (_used(case) + case["shared"]) * D * I * Q4_VALUE
    h = pairs * I * SIZE[case["h"]]
    if case["op"] == "gate_up":
        acts = n * D * SIZE[case["x"]] + h + 4 * n * top
    else:
        acts = h + 8 * n * top + 4 * n * case["shared"] + n * D * SIZE[case["y"]] * (1 + case["residual"])
    return {"bytes": weights + acts, "flops": 2 * matrices * pairs * D * I}


# -------------------------------------------------- the same in 64-bit torch

def _matrix64(w, s, b):
    """One quantized matrix [rows, words] in 64 bits, nibble or byte by its number of words."""
    cols = s.shape[-1] * 64
    bits = 32 * w.shape[-1] // cols
    parts = [(w >> (bits * i)) & ((1 << bits) - 1) for i in range(32 // bits)]
    q = torch.stack(parts, -1).reshape(w.shape[0], cols).double()
    return q * s.double().repeat_interleave(64, 1) + b.double().repeat_interleave(64, 1)


def _silu64(a):
    return a / (1 + torch.exp(-a))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        y = x / torch.sqrt((x * x).sum(1, keepdim=True) / case["cols"] + EPS) * s["w"].double()
        return [y, 1 / (1 + torch.exp(-(y @ _matrix64(*s["gate"])[0]))) if case["gate"] else None]
    if case["op"] == "sample":
        return _exact_sample(s)
    n, top = s["indices"].shape
    by_expert = [torch.nonzero(s["indices"] == e, as_tuple=True) for e in range(case["experts"])]
    if case["op"] == "gate_up":
        x = s["x"].double()
        out = torch.zeros(n, top + case["shared"], case["inter"], dtype=torch.float64, device=DEV)
        for e, (tok, slot) in enumerate(by_expert):
            if len(tok):
                Wg, Wu = (_matrix64(*(t[e] for t in s[k])) for k in ("gate", "up"))
                out[tok, slot] = _silu64(x[tok] @ Wg.t().contiguous()) * (x[tok] @ Wu.t().contiguous())
        if case["shared"]:
            Wg, Wu = _matrix64(*s["shared_gate"]), _matrix64(*s["shared_up"])
            out[:, top] = _silu64(x @ Wg.t().contiguous()) * (x @ Wu.t().contiguous())
        return out
    y = s["residual"].double() if case["residual"] else torch.zeros(n, case["hidden"], dtype=torch.float64, device=DEV)
    for e, (tok, slot) in enumerate(by_expert):
        if len(tok):
            W = _matrix64(*(t[e] for t in s["down"]))
            y[tok] += (s["h"][tok, slot].double() @ W.t().contiguous()) * s["scores"][tok, slot].double()[:, None]
    if case["shared"]:
        y += (s["h"][:, top].double() @ _matrix64(*s["shared_down"]).t().contiguous()) * s["coef"].double()[:, None]
    return y


def _exact_sample(s):
    """Row by row on the host, in the order that the filters are defined in."""
    tokens, probs = [], []
    rows = s["logits"].float().cpu().numpy().astype(np.float64)
    u, t, k, p, m = (s[name].cpu().numpy() for name in ("u", "temperature", "top_k", "top_p", "min_p"))
    for b in range(rows.shape[0]):
        l = rows[b]
        if not t[b] > 0:
            tokens.append(int(np.argmax(l)))
            probs.append(1.0)
            continue
        e = np.exp((l - l.max()) / np.float64(t[b]))
        order = np.argsort(-l, kind="stable")
        n = min(int(k[b]), len(l)) if k[b] > 0 else len(l)
        mass = np.rint(e * UNIT).astype(np.int64)
        cum = np.cumsum(mass[order[:n]])
        if p[b] < 1:
            n_p = int(np.searchsorted((cum - mass[order[:n]]).astype(np.float64), np.float64(p[b]) * np.float64(cum[-1]), side="left"))
        else:
            n_p = n
        n_m = int((e[order[:n]] >= np.float64(m[b])).sum()) if m[b] > 0 else n
        kept = np.sort(order[:max(1, min(n_p, n_m))])
        cum = np.cumsum(mass[kept])
        aim = min(int(np.floor(np.float64(u[b]) * np.float64(cum[-1]))), int(cum[-1]) - 1)
        at = int(np.searchsorted(cum, aim, side="right"))
        tokens.append(int(kept[at]))
        probs.append(float(mass[kept[at]]) / float(cum[-1]))
    return [torch.tensor(tokens, dtype=torch.int32, device=DEV), torch.tensor(probs, dtype=torch.float64, device=DEV)]
