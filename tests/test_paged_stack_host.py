"""The paged stack's own bookkeeping on the CPU: what it refuses, and that a
refused call leaves slots, lengths and pages as they were. No layer runs: the
context is a stand-in and the stacks have states but no layers to compute."""
import types

import pytest
import torch

from qff.pages import OutOfPages, PageTable
from qff.stack import AttentionStack

SLOTS, PAGE = 4, 16


def _ctx(max_batch=8, max_ctx=256, max_prefill_tokens=64, device=0):
    return types.SimpleNamespace(device=device, handle=None,
                                 cfg=types.SimpleNamespace(max_batch=max_batch, max_ctx=max_ctx, max_prefill_tokens=max_prefill_tokens))


def _stack(kinds=("dn", "gqa"), pages=12, ctx=None, max_ctx=256, slots=SLOTS):
    """A stack on the host whose slots' states and pools hold something."""
    table = PageTable(pages, PAGE, slots, max_ctx, device="cpu")
    states = []
    for kind in kinds:
        if kind == "dn":
            states.append({"conv_state": torch.randn(slots, 6, 4), "ssm_state": torch.randn(slots, 2, 8)})
        else:
            states.append({k: torch.randn(pages, PAGE, 2, 256).bfloat16() for k in ("k_pages", "v_pages")})
    return AttentionStack(ctx or _ctx(), [{}] * len(kinds), slots, max_ctx, states=states, kinds=kinds, device="cpu", pages=table)


def _snapshot(st):
    P = st.pages
    return (list(P.lengths), P.refs.copy().tolist(), sorted(P._free), P._rows.tolist(), P.table.tolist(), P.group.tolist(),
            P.shared_len.tolist(), [[t.clone() for t in S.values()] for S in st.states])


def _same(a, b):
    return a[:-1] == b[:-1] and all(torch.equal(x, y) for s, t in zip(a[-1], b[-1]) for x, y in zip(s, t))


@pytest.mark.parametrize("x", [torch.zeros(20, 2048), torch.zeros(20, 4096)[:, ::2], torch.zeros(2048, 20).t(),
                               torch.zeros(20, 2048, dtype=torch.bfloat16), torch.zeros(20, 2047), torch.zeros(2048),
                               torch.zeros(65, 2048), torch.zeros(0, 2048)])
def test_a_refused_slice_changes_nothing(x):
    """x on the host, in another layout, type or shape, too long, empty: the
    slot is as before, so a retry is not refused for what the first left."""
    st = _stack()
    before = _snapshot(st)
    with pytest.raises(ValueError):
        st.prefill(1, x)
    assert _same(before, _snapshot(st))


@pytest.mark.parametrize("x", [torch.zeros(20, 4096)[:, ::2], torch.zeros(2048, 20).t()])
def test_a_slice_in_another_layout_is_refused_on_its_device(x):
    """(The stand-in's device is the host here, so that only the layout is wrong.)"""
    st = _stack(ctx=_ctx(device=-1))
    before = _snapshot(st)
    with pytest.raises(ValueError, match="contiguous"):
        st.prefill(1, x)
    assert _same(before, _snapshot(st))


def test_a_table_that_the_context_cannot_serve_is_refused_at_once():
    for ctx, slots, match in ((_ctx(max_ctx=128), SLOTS, "max_ctx"), (_ctx(max_batch=3), SLOTS, "max_batch")):
        with pytest.raises(ValueError, match=match):
            _stack(ctx=ctx, slots=slots)
    table = PageTable(4, PAGE, SLOTS, 256, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        AttentionStack(_ctx(), [], SLOTS + 1, 256, states=[], kinds=[], device="cpu", pages=table)
    _stack(ctx=_ctx(max_ctx=250))    # 256 positions in whole pages
