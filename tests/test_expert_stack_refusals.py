"""What a stack with expert blocks and a head refuses, on the CPU: whatever one of its calls would refuse in the middle of
a step is refused when the stack is made or before the step's first layer, with every slot as it was."""
import types

import pytest
import torch

from qff.ops import ExpertWeights
from qff.pages import PageTable
from qff.stack import AttentionStack
from test_paged_host import on_host  # noqa: F401  (the fixture)
from test_paged_stack_host import PAGE, SLOTS, _ctx, _same, _snapshot

BF, F16 = torch.bfloat16, torch.float16


def _q(bits, *shape, sb=F16):
    *lead, cols = shape
    return (torch.zeros(*lead, cols * bits // 32, dtype=torch.int32), torch.zeros(*lead, cols // 64, dtype=sb),
            torch.zeros(*lead, cols // 64, dtype=sb))


def _mlp(E=8, I=64, row=_q(8, 1, 2048), **change):
    """(row: the shared expert's gate)"""
    experts = {"gate": _q(4, E, I, 2048), "up": _q(4, E, I, 2048), "down": _q(4, E, 2048, I), "shared_gate": _q(4, I, 2048),
               "shared_up": _q(4, I, 2048), "shared_down": _q(4, 2048, I)}
    experts.update({k: change.pop(k) for k in list(change) if k in experts})
    return {"norm_w": torch.ones(2048), "router": _q(8, E, 2048), "gate": row, "experts": ExpertWeights(**experts), **change}


def _stack(mlp, ctx=None, head=None, batch=SLOTS):
    """Two layers with states, the first recurrent, both with the block."""
    table = PageTable(12, PAGE, batch, 256, device="cpu")
    states = [{"conv_state": torch.randn(batch, 6, 4), "ssm_state": torch.randn(batch, 2, 8)},
              {k: torch.randn(12, PAGE, 2, 256).bfloat16() for k in ("k_pages", "v_pages")}]
    return AttentionStack(ctx or _ctx(), [{"mlp": mlp}] * 2, batch, 256, states=states, kinds=["dn", "gqa"], device="cpu", pages=table,
                          head=head)


@pytest.mark.parametrize("change,error,match", [
    ({"E": 264}, ValueError, "8 .. 256 experts"), ({"E": 4}, ValueError, "8 .. 256 experts"), ({"I": 4160}, ValueError, "4096 rows"),
    ({"router": _q(8, 8, 1024)}, ValueError, "router must be"), ({"router": (_q(8, 8, 2048)[0], *_q(8, 8, 1024)[1:])}, ValueError, "router: scales"),
    ({"router": _q(8, 8, 2048, sb=torch.float32)}, TypeError, "router: scales"),
    ({"row": _q(8, 2, 2048)}, ValueError, "gate must be"), ({"row": _q(8, 1, 1024)}, ValueError, "gate must be"),
    ({"norm_w": torch.ones(1024)}, ValueError, "norm_w must be"), ({"norm_w": torch.ones(2048).half()}, ValueError, "norm_w must be"),
    ({"up": _q(4, 8, 64, 1024)}, ValueError, "up must be"), ({"down": _q(4, 8, 2048, 64, sb=BF)}, TypeError, "one type"),
    ({"shared_down": _q(4, 2048, 128)}, ValueError, "shared_down must be")])
def test_a_block_that_a_call_would_refuse(change, error, match):
    with pytest.raises(error, match=match):
        _stack(_mlp(**change))


def test_a_head_that_a_call_would_refuse():
    norm = torch.ones(2048)
    for head, match in (({"norm_w": norm, "lm_head": _q(4, 128, 1024)}, "lm_head must be"), ({"norm_w": norm[:64], "lm_head": _q(4, 128, 2048)}, "norm_w must be"),
                        ({"norm_w": norm.half(), "lm_head": _q(4, 128, 2048)}, "norm_w must be"),
                        ({"norm_w": norm, "lm_head": tuple(t.expand(262145, -1) for t in _q(4, 1, 2048))}, "262144 rows"),
                        ({"norm_w": norm, "lm_head": (_q(4, 128, 2048)[0], *_q(4, 128, 1024)[1:])}, "lm_head: scales")):
        with pytest.raises(ValueError, match=match):
            _stack(None, head=head)
    ctx = types.SimpleNamespace(device=0, handle=None, cfg=types.SimpleNamespace(max_batch=2, max_ctx=64, max_prefill_tokens=8))
    for mlp, head in ((_mlp(), None), (None, {"norm_w": norm, "lm_head": _q(4, 128, 2048)})):
        with pytest.raises(ValueError, match="max_batch"):
            AttentionStack(ctx, [{"mlp": mlp}], 3, 64, kinds=["gqa"], device="cpu", head=head)


def _strided(q):
    return (torch.zeros(*q[0].shape, 2, dtype=torch.int32)[..., 0], *q[1:])


@pytest.mark.parametrize("change,match", [
    ({"down": _strided(_q(4, 8, 2048, 64))}, "down must be contiguous"), ({"shared_up": _strided(_q(4, 64, 2048))}, "shared_up must be contiguous"),
    ({"router": _strided(_q(8, 8, 2048))}, "router must be contiguous"), ({"row": _strided(_q(8, 1, 2048))}, "gate must be contiguous"),
    ({"norm_w": torch.ones(2048, 2)[:, 0]}, "norm_w must be contiguous")])
def test_a_block_that_lies_wrong_is_refused_before_anything_moves(on_host, change, match):  # noqa: F811
    """(The stand-in's device is the host here, so that only the layout is wrong.)"""
    ctx, calls = on_host
    ctx.cfg = _ctx().cfg
    st = _stack(_mlp(**change), ctx=ctx)
    st.pages.reserve(1, 0, 5)
    st.pages.sync()
    before = _snapshot(st)
    for _ in range(2):   # (and again, while it is wrong)
        for call in (lambda: st.prefill(0, torch.zeros(3, 2048)), lambda: st.reserve([-1, 5, -1, -1]),
                     lambda: st.decode_step(torch.zeros(SLOTS, 2048), torch.zeros(SLOTS, dtype=torch.int32))):
            with pytest.raises(ValueError, match=match):
                call()
            assert _same(before, _snapshot(st)) and not st._parked
    assert not {"qff_q4_norm_matmul_parts", "qff_deltanet_decode", "qff_deltanet_prefill"} & set(calls.made)


def test_weights_on_another_device(on_host):  # noqa: F811
    st = _stack(_mlp())   # (the context's device is a GPU, the tensors lie on the host)
    before = _snapshot(st)
    with pytest.raises(ValueError, match="context's device"):
        st.reserve([0, -1, -1, -1])
    assert _same(before, _snapshot(st))


def test_a_block_that_fits_is_looked_at_once(on_host):  # noqa: F811
    ctx, calls = on_host
    ctx.cfg = _ctx().cfg
    st = _stack(_mlp(), ctx=ctx)
    st.reserve([0, 0, -1, -1])
    assert calls.made == ["qff_rms_norm", "qff_moe_gate_up", "qff_moe_down"] * 2 and st.pages.lengths == [1, 1, 0, 0]
    st.reserve([1, 1, -1, -1])
    assert len(calls.made) == 6
    st = _stack(_mlp(row=None, shared_gate=None, shared_up=None, shared_down=None), ctx=ctx)
    st.reserve([0, -1, -1, -1])
    assert len(calls.made) == 12
