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


def _copy(st, monkeypatch):
    """The page copies of the stack, on the host."""
    def pages_copy(ctx, pools, src, dst):
        for pool in pools:
            for s, d in zip(src, dst):
                pool[d] = pool[s]
    monkeypatch.setattr("qff.stack.ops.pages_copy", pages_copy)


def _hold(st, slot, n):
    """Slot `slot` holds n positions, as a prompt's slices leave it."""
    st.pages.reserve(slot, 0, n)
    st.pages.sync()


@pytest.mark.parametrize("positions", [[20, -1, 7, -1], [20, -1, 4, -1], [20, -1, 5, 1], [20, -1, 5, 256], [20, 3, 5, -1]])
def test_a_step_follows_what_each_slot_holds(positions):
    """A position before the end would advance recurrent states twice, one past
    it leaves a hole: refused with no slot changed, the ones before it neither."""
    st = _stack()
    _hold(st, 0, 20)
    _hold(st, 2, 5)
    before = _snapshot(st)
    with pytest.raises(ValueError):
        st.reserve(positions)
    assert _same(before, _snapshot(st)) and not st._parked
    st.reserve([20, -1, 5, 0])
    assert st.pages.lengths == [21, 0, 6, 1]


def test_a_stack_without_recurrent_layers_may_go_back(monkeypatch):
    st = _stack(kinds=("gqa",))
    _copy(st, monkeypatch)
    _hold(st, 0, 20)
    st.reserve([18, -1, -1, -1])
    assert st.pages.lengths == [20, 0, 0, 0]


@pytest.mark.parametrize("kinds", [("dn", "gqa"), ("gqa",)])
def test_out_of_pages_takes_the_steps_positions_back(monkeypatch, kinds):
    """Slot 0 would begin a page, slot 1 copy a shared one, slot 2 find none
    free: none counts its position, and the same step goes through once there is
    room, with states as they were."""
    st = _stack(kinds=kinds, pages=4)
    _copy(st, monkeypatch)
    _hold(st, 0, 16)
    _hold(st, 1, 5)
    st.pages.fork(1, 2)
    st.pages.sync()
    states = [t.clone() for t in st._recurrent()]
    first = st.pages.pages_of(1)[0]
    _hold(st, 3, 2)                     # (one page is left)
    with pytest.raises(OutOfPages):
        st.reserve([16, 5, 5, -1])      # slot 0 takes it, slot 1 is refused
    assert st.pages.lengths == [16, 5, 5, 2] and st.pages.free_pages == 1
    assert [st.pages.pages_of(s) for s in (1, 2)] == [[first], [first]]
    st.reserve([-1, 5, -1, -1])         # sits out: the position it did not get is not counted
    assert st.pages.lengths == [16, 6, 5, 2]
    with pytest.raises(OutOfPages):
        st.reserve([16, 6, 5, -1])
    assert st.pages.lengths == [16, 6, 5, 2]
    st.release(3)
    st.reserve([16, 6, 5, -1])
    assert st.pages.lengths == [17, 7, 6, 0]
    assert all(torch.equal(a, b) for a, b in zip(states, st._recurrent()))


def test_a_sequence_that_could_not_begin_begins_later(monkeypatch):
    """Position 0 of an empty slot, taken back: the slot is empty again, and the
    next try begins with zero states."""
    st = _stack(pages=2)
    _copy(st, monkeypatch)
    _hold(st, 1, 16)
    with pytest.raises(OutOfPages):
        st.reserve([0, 16, -1, -1])
    assert st.pages.lengths == [0, 16, 0, 0] and st.pages.free_pages == 1
    st._recurrent()[0][0] = 7.0         # (what steps leave in a slot without a position)
    st.reserve([0, -1, -1, -1])
    assert all(not t[0].any() for t in st._recurrent())


@pytest.mark.parametrize("slot", [-1, -SLOTS, SLOTS])
def test_what_is_no_slots_number_is_refused(slot):
    """A negative number would be another slot's pages, and not its parked states."""
    st = _stack(ctx=_ctx(device=-1))
    _hold(st, 3, 40)
    before = _snapshot(st)
    P = st.pages
    for call in (lambda: st.prefill(slot, torch.zeros(4, 2048)), lambda: st.release(slot), lambda: st.fork(slot, [1]),
                 lambda: st.fork(3, [0, slot]), lambda: P.reserve(slot, 0, 1), lambda: P.release(slot), lambda: P.fork(slot, 0),
                 lambda: P.fork(3, slot), lambda: P.truncate(slot, 0), lambda: P.pages_of(slot)):
        with pytest.raises(IndexError):
            call()
        assert _same(before, _snapshot(st))


@pytest.mark.parametrize("positions,error", [(torch.zeros(SLOTS), TypeError), (torch.zeros(SLOTS, dtype=torch.int64), TypeError),
                                             (torch.zeros(SLOTS - 1, dtype=torch.int32), TypeError),
                                             (torch.zeros(2 * SLOTS, dtype=torch.int32)[::2], ValueError),
                                             (torch.zeros(SLOTS, dtype=torch.int32, device="meta"), ValueError)])
def test_a_step_is_refused_before_its_first_layer(monkeypatch, positions, error):
    """A full-attention layer behind recurrent ones would refuse these positions
    with the states before it advanced."""
    st = _stack(ctx=_ctx(device=-1))
    ran = []
    monkeypatch.setattr(st, "layer_step", lambda l, x, pos: ran.append(l))
    with pytest.raises(error):
        st.decode_step(torch.zeros(SLOTS, 2048), positions)
    assert not ran
    st.decode_step(torch.zeros(SLOTS, 2048), torch.zeros(SLOTS, dtype=torch.int32))
    assert ran == [0, 1]
