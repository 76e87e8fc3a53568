"""The expert block, the norm and sampling in 64 bits on the host, and how far fp32
sums of exact products may be from them."""
import numpy as np
import torch

U32 = 2.0 ** -24   # half a step of fp32, relative


def quantized(rng, shape, cols, bits, sb):
    """Random affine-quantized matrices [*shape, cols]: int32 words, scales and biases of type sb (torch, host)."""
    w = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (*shape, cols * bits // 32)).astype(np.int32))
    top = 2 ** bits - 1
    s = rng.uniform(0.5, 1.5, (*shape, cols // 64)) * 3.4 / top / np.sqrt(cols)
    b = -s * top / 2 + 0.3 / np.sqrt(cols) * rng.standard_normal(s.shape)
    return w, torch.from_numpy(s).to(sb), torch.from_numpy(b).to(sb)


def parts64(q, bits):
    """(nibbles or bytes, scales, biases), each [.., cols] in float64."""
    w, s, b = q
    v = w.numpy().view(np.uint32)
    per = 32 // bits
    nib = ((v[..., None] >> (bits * np.arange(per, dtype=np.uint32))) & (2 ** bits - 1)).reshape(*v.shape[:-1], -1)
    return nib.astype(np.float64), s.double().numpy().repeat(64, -1), b.double().numpy().repeat(64, -1)


def dense64(q, bits=4):
    nib, s, b = parts64(q, bits)
    return nib * s + b


def product(q, x, x_err, fp16=False):
    """x [n, cols] (float64) times one quantized matrix [rows, cols]: the product and a bound on the error of a kernel
    that sums exact products in fp32, x off by x_err [n, cols].

    fp32 sums: each group of 64 columns is summed in at most 6 matrix products (two k steps of three terms) of 32 products
    each, so a term passes at most 6 * 32 roundings there, then one for each of the G groups, at most 8 for the waves' sums
    and 2 for the scaling: 202 + G roundings of partial sums that are at most the sum of the terms' magnitudes, which are
    (16 + q) |s| |x| and |b - 16 s| |x| in the form that is summed.
    fp16: weights s (q - 8) rounded to fp16 (half a step 2^-11) where the scale has more than 8 bits."""
    nib, s, b = parts64(q, 4)
    W = nib * s + b
    G = W.shape[-1] // 64
    mag = (16 + nib) * np.abs(s) + np.abs(b - 16 * s)
    ax = np.abs(x)
    err = U32 * (202 + G) * (ax @ mag.T) + x_err @ np.abs(W).T
    if fp16:
        err += 2.0 ** -11 * (ax @ (np.abs(nib - 8) * np.abs(s)).T)
    return x @ W.T, err


def silu64(a):
    return a / (1 + np.exp(-a))


HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# (half a step of each type, relative: bf16 has an eps of 2^-7, fp16 of 2^-10)
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}   # half a step of fp16's subnormals


def gate_up(gate, up, shared_gate, shared_up, x, indices, x_err=None, fp16=False):
    """h [n, slots, inter] and a bound on its fp32 error; rows of indices that are no expert's are NaN."""
    E = gate[0].shape[0]
    n, top = indices.shape
    x_err = np.zeros_like(x) if x_err is None else x_err
    h = np.full((n, top + (shared_gate is not None), gate[0].shape[1]), np.nan)
    err = np.zeros_like(h)

    def fill(where, g, u):
        (g, eg), (u, eu) = g, u
        # |silu'| <= 1.1; expf, the quotient and the product: 8 roundings at most
        h[where] = silu64(g) * u
        err[where] = 1.1 * eg * np.abs(u) + np.abs(silu64(g)) * eu + 1.1 * eg * eu + 8 * U32 * np.abs(silu64(g) * u)

    for e in range(E):
        tok, slot = np.nonzero(indices == e)
        if len(tok):
            g, u = ([t[e] for t in m] for m in (gate, up))
            fill((tok, slot), product(g, x[tok], x_err[tok], fp16), product(u, x[tok], x_err[tok], fp16))
    if shared_gate is not None:
        fill((np.arange(n), top), product(shared_gate, x, x_err, fp16), product(shared_up, x, x_err, fp16))
    return h, err


def down(w, shared, h, indices, scores, coef, residual, h_err=None, fp16=False, part=0.0):
    """y [n, hidden] and a bound on its fp32 error; `part`: what a pair's row is rounded by on the way, relative to its
    largest entry."""
    E, D = w[0].shape[:2]
    n, top = indices.shape
    y = np.zeros((n, D)) if residual is None else residual.astype(np.float64).copy()
    mag, err = np.abs(y), np.zeros((n, D))

    def add(m, q, rows, rows_err, f):
        p, e = product(q, rows, rows_err, fp16)
        f = np.abs(f)[:, None]
        np.add.at(err, m, f * (e + 2 * U32 * np.abs(p) + part * np.abs(p).max(1, keepdims=True)))
        np.add.at(mag, m, f * np.abs(p))
        return p

    for e in range(E):
        tok, slot = np.nonzero(indices == e)
        if len(tok):
            f = scores[tok, slot]
            p = add(tok, [t[e] for t in w], h[tok, slot], np.zeros_like(h[tok, slot]) if h_err is None else h_err[tok, slot], f)
            np.add.at(y, tok, f[:, None] * p)
    if shared is not None:
        f = np.ones(n) if coef is None else coef
        p = add(np.arange(n), shared, h[:, top], np.zeros_like(h[:, top]) if h_err is None else h_err[:, top], f)
        y += f[:, None] * p
    # the sum over the slots (or, for few pairs, over the waves that share them) and the residual
    return y, err + (top + 12) * U32 * mag


def within(got, ref, err, dtype):
    """Whether got (of `dtype`, as float64) is ref's rounding, ref known to err."""
    return np.abs(got - ref) <= HALF[dtype] * (np.abs(ref) + err) + err + LEAST[dtype]


UNIT = 2.0 ** 44


def sample_row(l, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, chance) of one row of logits by the definition, filter by filter."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    t, p, m, u = (float(np.float32(v)) for v in (t, p, m, u))
    if l.max() == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(l)), 1.0
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.exp((l - l.max()) / t)
    e[l == l.max()] = 1.0
    e[(l == -np.inf) | np.isnan(e)] = 0.0
    mass = [int(v) for v in np.rint(e * UNIT)]
    order = sorted(range(len(l)), key=lambda i: (-l[i], i))
    head = order[:k] if k > 0 else order
    weight, before, kept = sum(mass[i] for i in head), 0, []
    for i in head:
        if p < 1 and not float(before) < p * float(weight):
            break
        if m > 0 and not e[i] >= m:
            break
        kept.append(i)
        before += mass[i]
    kept = sorted(kept or order[:1])
    total = sum(mass[i] for i in kept)
    aim = min(int(np.floor(min(max(u, 0.0), 1.0) * float(total))), total - 1)
    run = 0
    for i in kept:
        run += mass[i]
        if run > aim:
            return i, mass[i] / total
