"""The expert block at the ends of what its weights may hold, and between them, in every form. Rows of x (or h) with one column that is not 0 make every output a single weight times x: a few
roundings, so that a bound is sharp enough to show a part that a kernel lost."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV
from test_gpu_moe import DT, _ctx, _indices, _np64, _to

pytestmark = pytest.mark.gpu

# (tokens, experts, top): each pair by itself, small tiles, and large ones of 32, 64 and 128 pairs (x or h in one term; in
# two, the last ones are of 64)
FORMS = {"one": (2, 3, 2), "slim": (70, 200, 4), "tile32": (80, 4, 1), "tile64": (80, 2, 1), "tile128": (150, 2, 1)}
# (down takes more pairs one by one)
DOWN_FORMS = {"one": (2, 3, 2), "slim": (70, 200, 4), "tile32": (210, 10, 1), "tile64": (210, 7, 1), "tile128": (210, 3, 1)}


def _bits(rng, shape, lo, hi, bits):
    """Numbers of both signs with `bits` significant bits, spread over the logarithm of lo .. hi (lo the power of two below)."""
    e = rng.integers(int(np.floor(np.log2(lo))), int(np.floor(np.log2(hi))) + 1, shape)
    m = 1 + rng.integers(0, 2 ** (bits - 1), shape) / 2.0 ** (bits - 1)
    return np.minimum(m * 2.0 ** e, hi) * rng.choice([-1.0, 1.0], shape)


def _extreme(rng, shape, cols, sb, end):
    """Affine-Q4 matrices whose scales lie at one end of 2^-22 .. 31 (or 0), |bias + 8 scale| up to 8."""
    w = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (*shape, cols // 8)).astype(np.int32))
    g = (*shape, cols // 64)
    if end == "large":
        s = rng.choice([31.0, 30.875, 24.0, 16.125, 10.75, 10.5], g) * rng.choice([-1.0, 1.0], g)
        c = rng.choice([0.0, 1.0, -3.0, 7.0, 8.0, -8.0], g)
    elif end == "usual":   # neither end, scales of all the bits that their type has
        s, c = (_bits(rng, g, lo, hi, 8 if sb == "bf16" else 11) for lo, hi in ((2.0 ** -8, 2.0 ** -6), (2.0 ** -6, 2.0 ** -3)))
    elif end == "parts":   # the constant parts alone: every nibble 8
        w.fill_(-2004318072)
        s = rng.choice([0.0, 1.0, 2.0 ** -10, 2.0 ** -20], g)
        c = np.where(s == 1.0, 8.0, _bits(rng, g, 2.0 ** -22, 8.0, 8))
        c = np.where(s == 0.0, rng.choice([8.0, -8.0, 7.75, 2.0 ** -20], g), c)
    elif end == "small parts":   # alone, and far below the smallest scale
        w.fill_(-2004318072)
        s, c = np.zeros(g), _bits(rng, g, 2.0 ** -34, 2.0 ** -30, 8)
    else:
        s = _bits(rng, g, 2.0 ** -22, 2.0 ** -20, 8 if sb == "bf16" else 3)   # (fp16 ends at 2^-24)
        c = _bits(rng, g, 2.0 ** -22, 2.0 ** -19, 4)
    s = torch.from_numpy(s).to(DT[sb])
    b = (torch.from_numpy(c) - 8 * s.double()).to(DT[sb])
    part = (b.double() + 8 * s.double()).abs()
    b = torch.where(part <= 8, b.double(), -8 * s.double()).to(DT[sb])   # (where the rounding took it past 8)
    assert ((b.double() + 8 * s.double()).abs() <= 8).all() and (s.abs() <= 31).all()
    return w, s, b


def _one_column(rng, shape, cols, size):
    """[*shape, cols] with one value of 24 bits a row."""
    x = np.zeros((*shape, cols), np.float32)
    v = (size * rng.uniform(0.5, 1.0, shape) * rng.choice([-1.0, 1.0], shape)).astype(np.float32)
    np.put_along_axis(x, rng.integers(0, cols, (*shape, 1)), v[..., None], -1)
    return torch.from_numpy(x)


def _single(q, x, x_terms, w_terms):
    """x [n, cols] with one column a row times one matrix, and a bound on the error. The form of single pairs: (16 + q) |s|
    and |b - 16 s| cancel, 16 roundings. The others: s (q - 8), exact in two terms, and c = b + 8 s in 22 bits, against x and
    its groups' sums in two terms of 11 bits (one term: 11 bits of x, of the product s (q - 8) for one of the weight):
    2^-22 for each term's rest, for the products of both rests and for c, and 16 roundings."""
    nib, s, b = R.parts64(q, 4)
    W, c, ax = nib * s + b, b + 8 * s, np.abs(x)
    main, const = np.abs(nib - 8) * np.abs(s), np.abs(c)
    if x_terms == 0:
        return x @ W.T, 16 * R.U32 * (ax @ ((16 + nib) * np.abs(s) + np.abs(b - 16 * s)).T)
    err = (4 * 2.0 ** -22 + 16 * R.U32) * (ax @ (main + const).T) + 2.0 ** -46 * ax.sum(-1, keepdims=True)
    if x_terms == 1:
        err += 2.0 ** -11 * (ax @ main.T)
    if w_terms == 1:
        err += 2.0 ** -11 * (ax @ main.T)
    return x @ W.T, err


def _rounded_within(got, ref, err, dtype):
    """got is the rounding to `dtype` of a number within err of ref."""
    lo, hi = ((torch.from_numpy(v).to(dtype).double().numpy() for v in (ref - err, ref + err)))
    ok = (got >= lo) & (got <= hi)
    assert ok.all(), f"{(~ok).sum()} of {ok.size} outside; {got[~ok][:4]} instead of {ref[~ok][:4]}"


def _terms(form, dtype, sb, out):
    """Terms of x and of a weight that a form keeps (0: exact)."""
    if form == "one":
        return 0, 0
    all_terms = out != "bf16"
    return (2 if dtype != "f32" or all_terms else 1), (2 if sb == "bf16" or all_terms else 1)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("end", ["parts", "small parts", "large", "small", "usual"])
@pytest.mark.parametrize("x_dt,h_dt,sb", [("f32", "f32", "bf16"), ("f32", "f16", "f16"), ("bf16", "f32", "f16"), ("f32", "bf16", "bf16"),
                                          ("bf16", "bf16", "f16")])
def test_gate_up_at_the_ends(hip, form, end, x_dt, h_dt, sb):
    import qff
    print(f"gate_up ends {form} {end} x={x_dt} h={h_dt} sb={sb}", flush=True)
    n, E, top = FORMS[form]
    D, I = 192, 128
    rng = np.random.default_rng(len(form) + 10 * len(end))
    gate, up = (_extreme(rng, (E, I), D, sb, end) for _ in range(2))
    x = _one_column(rng, (n,), D, {"large": 2.0 ** -6, "small": 2.0 ** 20, "parts": 0.5, "small parts": 2.0 ** 20, "usual": 32.0}[end]).to(DT[x_dt])
    idx = _indices(rng, n, E, top, "any")
    got = _np64(qff.moe_gate_up(_ctx(), qff.ExpertWeights(_to(gate), _to(up)), x.to(DEV), torch.from_numpy(idx).to(DEV), out_dtype=DT[h_dt]))
    x64, terms = x.double().numpy(), _terms(form, x_dt, sb, h_dt)
    ref, err = np.zeros(got.shape), np.zeros(got.shape)
    for e in range(E):
        tok, slot = np.nonzero(idx == e)
        if len(tok):
            (g, eg), (u, eu) = (_single([t[e] for t in m], x64[tok], *terms) for m in (gate, up))
            ref[tok, slot] = R.silu64(g) * u
            # |silu'| <= 1.1; expf, the quotient and the product: 8 roundings
            err[tok, slot] = 1.1 * eg * np.abs(u) + np.abs(R.silu64(g)) * eu + 1.1 * eg * eu + 8 * R.U32 * np.abs(R.silu64(g) * u)
    _rounded_within(got, ref, err, DT[h_dt])


@pytest.mark.parametrize("form", DOWN_FORMS)
@pytest.mark.parametrize("end", ["parts", "small parts", "large", "small", "usual"])
@pytest.mark.parametrize("h_dt,y_dt,sb", [("f32", "f32", "f16"), ("f16", "f32", "bf16"), ("bf16", "f32", "f16"), ("f32", "bf16", "bf16"),
                                          ("f16", "bf16", "f16")])
def test_down_at_the_ends(hip, form, end, h_dt, y_dt, sb):
    import qff
    print(f"down ends {form} {end} h={h_dt} y={y_dt} sb={sb}", flush=True)
    n, E, top = DOWN_FORMS[form]
    D, I = 128, 192
    rng = np.random.default_rng(len(form) + 10 * len(end))
    w = _extreme(rng, (E, D), I, sb, end)
    h = _one_column(rng, (n, top), I, 2.0 ** -4).to(DT[h_dt])
    idx = _indices(rng, n, E, top, "any")
    sc = (0.5 + rng.random((n, top))).astype(np.float32)
    got = _np64(qff.moe_down(_ctx(), qff.ExpertWeights(down=_to(w)), h.to(DEV), torch.from_numpy(idx).to(DEV), torch.from_numpy(sc).to(DEV),
                             out_dtype=DT[y_dt]))
    h64, terms = h.double().numpy(), _terms(form, h_dt, sb, y_dt)
    half = y_dt == "bf16" and form.startswith("tile")
    ref, err = np.zeros(got.shape), np.zeros(got.shape)
    for e in range(E):
        tok, slot = np.nonzero(idx == e)
        if len(tok):
            p, ep = _single([t[e] for t in w], h64[tok, slot], *terms)
            f = sc[tok, slot].astype(np.float64)[:, None]
            np.add.at(ref, tok, f * p)
            # a pair's row between the products and their sum: 11 bits of each value (and 2^-39 of the largest of 64)
            np.add.at(err, tok, f * (ep + 4 * R.U32 * np.abs(p) + half * (2.0 ** -11 * (np.abs(p) + ep) + 2.0 ** -39 * np.abs(p).max())))
    _rounded_within(got, ref, err + 8 * R.U32 * np.abs(ref), DT[y_dt])
