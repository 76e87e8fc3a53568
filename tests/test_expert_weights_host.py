"""The handle of a layer's expert weights on the host: tensors that move after its first call."""
import types

import pytest
import torch

from test_moe_host import D, E, _down_args, _up_args, _weights
from test_paged_host import on_host  # noqa: F401  (the fixture)


def test_weights_that_moved_are_read_where_they_lie_now(on_host, monkeypatch):  # noqa: F811
    """Tensors whose storage is replaced behind the first call's back: each call passes on the addresses of its own time,
    and checks what it has not seen."""
    import qff
    from qff import _lib, ops
    ctx, calls = on_host
    seen = []
    monkeypatch.setattr(ops, "_hot", lambda: types.SimpleNamespace(
        qff_moe_gate_up=lambda *a: seen.append(_lib.MoeWeights.from_buffer_copy(a[2])) or 0,
        qff_moe_down=lambda *a: seen.append(_lib.MoeWeights.from_buffer_copy(a[2])) or 0))
    w = _weights()
    gate, _, down, _, shared_up, shared_down = w.matrices
    up, dn = lambda: qff.moe_gate_up(ctx, **_up_args(experts=w)), lambda: qff.moe_down(ctx, **_down_args(experts=w))  # noqa: E731
    for call, t, field in ((up, gate[0], lambda s: s.gate.w), (up, shared_up[2], lambda s: s.shared_up.biases),
                           (dn, down[1], lambda s: s.down.scales), (dn, shared_down[0], lambda s: s.shared_down.w)):
        call()
        assert field(seen[-1]) == t.data_ptr()
        before = t.data_ptr()
        t.set_(t.clone())
        assert t.data_ptr() != before
        call()
        assert field(seen[-1]) == t.data_ptr()
        t.data = t.clone()
        call()
        assert field(seen[-1]) == t.data_ptr()
    # a smaller tensor in the old one's place is refused, and again
    n = len(seen)
    down[0].set_(torch.zeros(E, D, 1, dtype=torch.int32))
    for _ in range(2):
        with pytest.raises(ValueError, match="down: scales and biases"):
            dn()
    # gate and up too: what is wrong with a handle, every call says
    with pytest.raises(ValueError, match="down: scales and biases"):
        up()
    assert len(seen) == n
