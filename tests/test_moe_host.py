"""The expert block and sampling on the host, without a GPU: what the library
refuses (tests/host_checks/moe_checks.cpp), what the torch wrappers check
before they reach it, and the parameter blocks."""
import ctypes
import os
import subprocess
import types

import numpy as np
import pytest
import torch

import moe_ref as R
from test_paged_host import _program, on_host  # noqa: F401  (the fixture)


def test_library_refusals(tmp_path):
    import qff
    qff.lib()
    r = subprocess.run([_program(tmp_path, "moe_checks")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:]


def test_blocks_match_the_header(tmp_path):
    from qff import _lib, ops
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "qff/qff.h"', "int main(void) {"]
    mirrors = {"qff_q4_matrices": _lib.Q4Matrices, "qff_moe_weights": _lib.MoeWeights}
    for c, py in mirrors.items():
        lines.append(f'    printf("%zu\\n", sizeof({c}));')
        lines += [f'    printf("%zu\\n", offsetof({c}, {n}));' for n, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["    return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    want = [v for py in mirrors.values() for v in (ctypes.sizeof(py), *(getattr(py, n).offset for n, _ in py._fields_))]
    assert [int(v) for v in got] == want
    block = ops._P_MOE.pack(*range(1, 19), 1, 2, 3, 4)
    s = _lib.MoeWeights.from_buffer_copy(block)
    assert (s.gate.w, s.up.w, s.down.w, s.shared_gate.w, s.shared_up.w, s.shared_down.biases) == (1, 4, 7, 10, 13, 18)
    assert (s.sb_dtype, s.experts, s.hidden, s.inter) == (1, 2, 3, 4)


BF = torch.bfloat16
E, D, I = 3, 128, 64


def _q4(*shape, sb=BF):
    cols = shape[-1]
    return (torch.zeros(*shape[:-1], cols // 8, dtype=torch.int32), torch.ones(*shape[:-1], cols // 64, dtype=sb),
            torch.ones(*shape[:-1], cols // 64, dtype=sb))


def _weights(**change):
    import qff
    w = {"gate": _q4(E, I, D), "up": _q4(E, I, D), "down": _q4(E, D, I), "shared_gate": _q4(I, D), "shared_up": _q4(I, D),
         "shared_down": _q4(D, I)}
    return qff.ExpertWeights(**{**w, **change})


def _up_args(n=2, **change):
    return {"experts": _weights(), "x": torch.zeros(n, D), "indices": torch.zeros(n, 2, dtype=torch.int32), **change}


def _down_args(n=2, **change):
    return {"experts": _weights(), "h": torch.zeros(n, 3, I), "indices": torch.zeros(n, 2, dtype=torch.int32),
            "scores": torch.zeros(n, 2), **change}


def test_wrappers_pass_on_what_they_check(on_host):  # noqa: F811
    import qff
    ctx, calls = on_host
    for n in (0, 2):
        assert qff.moe_gate_up(ctx, **_up_args(n)).shape == (n, 3, I)
        assert qff.moe_down(ctx, **_down_args(n), coef=torch.zeros(n)).shape == (n, D)
        assert qff.rms_norm(ctx, torch.zeros(n, D), torch.ones(D)).shape == (n, D)
    gate = (torch.zeros(1, D // 4, dtype=torch.int32), torch.ones(1, D // 64, dtype=BF), torch.ones(1, D // 64, dtype=BF))
    y, coef = qff.rms_norm(ctx, torch.zeros(2, D, dtype=BF), torch.ones(D), gate=gate, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and coef.shape == (2,)
    tok, prob = qff.sample(ctx, torch.zeros(2, 10), torch.zeros(2), top_k=torch.zeros(2, dtype=torch.int32))
    assert tok.dtype == torch.int32 and prob.shape == (2,)
    no = _weights(shared_gate=None, shared_up=None, shared_down=None)
    assert qff.moe_gate_up(ctx, **_up_args(experts=no)).shape == (2, 2, I)
    # a handle of one half's matrices alone
    assert qff.moe_gate_up(ctx, **_up_args(experts=_weights(down=None, shared_down=None))).shape == (2, 3, I)
    assert qff.moe_down(ctx, **_down_args(experts=_weights(gate=None, up=None, shared_gate=None, shared_up=None))).shape == (2, D)
    assert set(calls.made) == {"qff_rms_norm", "qff_moe_gate_up", "qff_moe_down", "qff_sample"}


@pytest.mark.parametrize("change,match", [
    ({"gate": None}, "gate and up come together"), ({"up": None}, "gate and up come together"),
    ({"shared_up": None}, "gate and up come together"), ({"shared_down": None}, "all three"),
    ({"shared_gate": None, "shared_up": None}, "all three"),
    ({"down": None}, "stand beside"), ({"gate": None, "up": None}, "stand beside"),
    ({"gate": None, "up": None, "down": None, "shared_gate": None, "shared_up": None, "shared_down": None}, "either"),
    ({"gate": _q4(I, D)}, "experts, rows")])
def test_handles_that_make_no_sense(change, match):
    with pytest.raises(ValueError, match=match):
        _weights(**change)


@pytest.mark.parametrize("change,error,match", [
    ({"up": _q4(E, I, 192)}, ValueError, "up must be"), ({"up": _q4(E + 1, I, D)}, ValueError, "up must be"),
    ({"down": _q4(E, I, D)}, ValueError, "down must be"), ({"shared_down": _q4(D, 128)}, ValueError, "shared_down must be"),
    ({"shared_up": _q4(1, I, D)}, ValueError, "shared_up must be"),
    ({"up": _q4(E, I, D, sb=torch.float16)}, TypeError, "one type"),
    ({"up": (_q4(E, I, D)[0], _q4(E, I, D)[1], _q4(E, I, D, sb=torch.float16)[2])}, TypeError, "up: scales and biases"),
    ({"up": _q4(E, I, D, sb=torch.float32)}, TypeError, "one type"),
    ({"gate": (_q4(E, I, D)[0].long(), *_q4(E, I, D)[1:])}, TypeError, "gate: the words"),
    ({"gate": (_q4(E, I, D)[0], _q4(E, I, 192)[1], _q4(E, I, D)[2])}, ValueError, "gate: scales and biases must be"),
    ({"gate": (_q4(E, I, D)[0], _q4(E, I, D)[1], _q4(E, I, 192)[2])}, ValueError, "gate: scales and biases must be"),
    ({"gate": (torch.zeros(E, I, 2 * D // 8, dtype=torch.int32)[:, :, ::2], *_q4(E, I, D)[1:])}, ValueError, "gate must be contiguous"),
    ({"down": (_q4(E, D, I)[0], torch.ones(E, D, 2, dtype=BF)[:, :, ::2], _q4(E, D, I)[2])}, ValueError, "down's scales must be contiguous")])
def test_weights_are_checked_by_the_first_call(on_host, change, error, match):  # noqa: F811
    import qff
    ctx, calls = on_host
    w = _weights(**change)
    for _ in range(2):   # (and by the next one, while they are wrong)
        with pytest.raises(error, match=match):
            qff.moe_gate_up(ctx, **_up_args(experts=w))
        with pytest.raises(error, match=match):
            qff.moe_down(ctx, **_down_args(experts=w))
    assert not calls.made


I32 = torch.int32


@pytest.mark.parametrize("change,error,match", [
    ({"x": torch.zeros(2, 64)}, ValueError, "x must be"), ({"x": torch.zeros(2, 1, D)}, ValueError, "x must be"),
    ({"x": torch.zeros(2, 2 * D)[:, ::2]}, ValueError, "x must be contiguous"),
    ({"x": torch.zeros(2, D, dtype=torch.float64)}, TypeError, "unsupported dtype"),
    ({"indices": torch.zeros(3, 2, dtype=I32)}, ValueError, "indices must be"), ({"indices": torch.zeros(2, dtype=I32)}, ValueError, "indices must be"),
    ({"indices": torch.zeros(2, 2, dtype=torch.int64)}, TypeError, "indices must be"),
    ({"indices": torch.zeros(2, 4, dtype=I32)[:, ::2]}, ValueError, "indices must be contiguous"),
    ({"out": torch.zeros(2, 2, I)}, ValueError, "out must be"), ({"out": torch.zeros(2, 3, 2 * I)[:, :, ::2]}, ValueError, "out must be contiguous")])
def test_gate_up_checks(on_host, change, error, match):  # noqa: F811
    import qff
    ctx, calls = on_host
    with pytest.raises(error, match=match):
        qff.moe_gate_up(ctx, **_up_args(**change))
    assert not calls.made


@pytest.mark.parametrize("change,error,match", [
    ({"h": torch.zeros(2, 2, I)}, ValueError, "h must be"), ({"h": torch.zeros(2, 3, 128)}, ValueError, "h must be"),
    ({"h": torch.zeros(2, 3, 2 * I)[:, :, ::2]}, ValueError, "h must be contiguous"),
    ({"indices": torch.zeros(1, 2, dtype=I32)}, ValueError, "indices must be"),
    ({"scores": torch.zeros(2, 3)}, ValueError, "scores must be"), ({"scores": torch.zeros(2, 2, dtype=BF)}, TypeError, "scores must be"),
    ({"coef": torch.zeros(3)}, ValueError, "coef must be"), ({"coef": torch.zeros(2, dtype=BF)}, TypeError, "coef must be"),
    ({"residual": torch.zeros(2, D, dtype=BF)}, ValueError, "a residual must match"), ({"residual": torch.zeros(1, D)}, ValueError, "a residual must match"),
    ({"residual": torch.zeros(2, 2 * D)[:, ::2]}, ValueError, "residual must be contiguous"),
    ({"out": torch.zeros(2, 64)}, ValueError, "out must be"), ({"out": torch.zeros(D, 2).t()}, ValueError, "out must be contiguous")])
def test_down_checks(on_host, change, error, match):  # noqa: F811
    import qff
    ctx, calls = on_host
    with pytest.raises(error, match=match):
        qff.moe_down(ctx, **_down_args(**change))
    assert not calls.made


def test_norm_and_sample_checks(on_host):  # noqa: F811
    import qff
    ctx, calls = on_host
    x, w = torch.zeros(2, D), torch.ones(D)
    g = (torch.zeros(1, D // 4, dtype=I32), torch.ones(1, D // 64, dtype=BF), torch.ones(1, D // 64, dtype=BF))
    for args, kw, error, match in (
            ((x, torch.ones(64)), {}, ValueError, "norm_w have cols"), ((x[0], w), {}, ValueError, "x must be"),
            ((x, w), {"out": torch.zeros(2, 64)}, ValueError, "out must be"), ((x.t(), torch.ones(2)), {}, ValueError, "x must be contiguous"),
            ((x, w), {"gate": (g[0][:, :16], *g[1:])}, ValueError, "gate: scales and biases|gate must be"),
            ((x, w), {"gate": tuple(t.repeat(2, 1) for t in g)}, ValueError, "gate must be"),
            ((x, w), {"gate": g, "coef": torch.zeros(1)}, ValueError, "coef must be"),
            ((x, w), {"gate": g, "coef": torch.zeros(2, dtype=BF)}, TypeError, "coef must be"),
            ((x.double(), w), {}, TypeError, "unsupported dtype")):
        with pytest.raises(error, match=match):
            qff.rms_norm(ctx, *args, **kw)
    l, u = torch.zeros(2, 10), torch.zeros(2)
    for args, kw, error, match in (
            ((l[0], u), {}, ValueError, "logits must be"), ((l, torch.zeros(3)), {}, ValueError, "u must be"),
            ((l, None), {}, TypeError, "u must be"), ((l, u.double()), {}, TypeError, "u must be"), ((l.double(), u), {}, TypeError, "unsupported"),
            ((l.t(), torch.zeros(10)), {}, ValueError, "logits must be contiguous"),
            ((l, u), {"temperature": torch.zeros(1)}, ValueError, "temperature must be"), ((l, u), {"top_k": torch.zeros(2)}, TypeError, "top_k must be"),
            ((l, u), {"top_p": torch.zeros(2, dtype=BF)}, TypeError, "top_p must be"), ((l, u), {"min_p": torch.zeros(3)}, ValueError, "min_p must be"),
            ((l, u), {"out": torch.zeros(2, dtype=torch.int64)}, TypeError, "out must be"), ((l, u), {"prob": torch.zeros(1)}, ValueError, "prob must be")):
        with pytest.raises(error, match=match):
            qff.sample(ctx, *args, **kw)
    assert not calls.made
    # tensors of another device than the context's
    other = types.SimpleNamespace(device=0, handle=None)
    for call in (lambda: qff.rms_norm(other, x, w), lambda: qff.sample(other, l, u), lambda: qff.moe_gate_up(other, **_up_args()),
                 lambda: qff.moe_down(other, **_down_args())):
        with pytest.raises(ValueError, match="context's device"):
            call()
    assert not calls.made


def test_sampling_definition():
    """The reference's own filters on a row whose weights are easy to say."""
    l = np.log(np.array([0.5, 0.25, 0.125, 0.125], np.float32))
    assert [R.sample_row(l, u)[0] for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.999)] == [0, 0, 1, 1, 2, 3]
    assert [R.sample_row(l, u, k=2)[0] for u in (0.6, 0.7)] == [0, 1]
    assert R.sample_row(l, 0.99, p=0.5) == (0, 1.0)         # nothing weighs before the first; half before the second is not less
    assert R.sample_row(l, 0.99, p=0.51)[0] == 1
    assert R.sample_row(l, 0.99, m=0.3)[0] == 1
    assert R.sample_row(l, 0.99, t=0.0) == (0, 1.0)
    assert R.sample_row(np.full(4, -np.inf), 0.5) == (-1, 0.0)
