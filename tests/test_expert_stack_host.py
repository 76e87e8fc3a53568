"""The expert block and the head of a stack on the CPU: what a checkpoint's
tensors become (parity unpinned: no file of the reference holds the experts'
names), and what a stack refuses. No layer runs."""
import os
import types

import numpy as np
import pytest
import torch

from ckpt_util import _q4, write_safetensors
from qff import synth
from qff.checkpoint import Checkpoint
from qff.ops import ExpertWeights
from qff.stack import AttentionStack

E, I = 8, 64


def _write(directory, shared=True, lm_head=True):
    rng = np.random.default_rng(3)
    pre, t = "language_model.model.", {}
    p = pre + "layers.1."
    for n, rows, cols in (("gate", I, 2048), ("up", I, 2048), ("down", 2048, I)):
        w, s, b = synth.q4_weight(E * rows, cols, seed=rows + len(n), sb_dtype="bf16")
        for part, a, dt in (("weight", w, "U32"), ("scales", s, "BF16"), ("biases", b, "BF16")):
            t[p + f"mlp.switch_mlp.{n}_proj.{part}"] = (a.reshape(E, rows, -1), dt)
        if shared:
            _q4(t, p + f"mlp.shared_expert.{n}_proj", rows, cols, seed=rows + 7)
    for stem, rows in (("mlp.gate", E), ("mlp.shared_expert_gate", 1))[:2 if shared else 1]:
        for part, a, dt in zip(("weight", "scales", "biases"), synth.q8_weight(rows, 2048, seed=rows), ("U32", "BF16", "BF16")):
            t[p + f"{stem}.{part}"] = (a, dt)
    norm = synth._bf16_bits(1 + 0.1 * rng.standard_normal(2048).astype(np.float32))
    t[p + "post_attention_layernorm.weight"] = (norm, "BF16")
    t[pre + "norm.weight"] = (norm, "BF16")
    _q4(t, "language_model.lm_head" if lm_head else pre + "embed_tokens", 128, 2048, seed=5)
    write_safetensors(os.path.join(directory, "model.safetensors"), t)
    return t


@pytest.mark.parametrize("shared", [True, False])
def test_expert_layer(tmp_path, shared):
    t = _write(tmp_path, shared)
    ck = Checkpoint(str(tmp_path))
    assert ck.expert_layer(0, "cpu") is None
    M = ck.expert_layer(1, "cpu")
    W = M["experts"]
    assert (W.experts, W.hidden, W.inter, W.dtype) == (E, 2048, I, torch.bfloat16)
    p = "language_model.model.layers.1.mlp."
    for q, stem in zip(W.matrices, [f"switch_mlp.{n}_proj" for n in ("gate", "up", "down")] +
                       [f"shared_expert.{n}_proj" for n in ("gate", "up", "down")]):
        if q is None:
            assert not shared
            continue
        assert np.array_equal(q[0].numpy().view(np.uint32), t[p + stem + ".weight"][0])
        assert np.array_equal(q[2].view(torch.int16).numpy().view(np.uint16), t[p + stem + ".biases"][0])
    assert (M["gate"] is None) == (not shared) and M["router"][0].shape == (E, 512)
    assert M["norm_w"].dtype == torch.float32
    ck.close()


@pytest.mark.parametrize("lm_head", [True, False])
def test_head(tmp_path, lm_head):
    t = _write(tmp_path, lm_head=lm_head)
    ck = Checkpoint(str(tmp_path))
    H = ck.head("cpu")
    stem = "language_model.lm_head" if lm_head else "language_model.model.embed_tokens"
    assert np.array_equal(H["lm_head"][0].numpy().view(np.uint32), t[stem + ".weight"][0]) and H["norm_w"].shape == (2048,)
    ck.close()


def _q(rows, cols, experts=None):
    lead = (rows,) if experts is None else (experts, rows)
    return (torch.zeros(*lead, cols // 8, dtype=torch.int32), torch.zeros(*lead, cols // 64).half(), torch.zeros(*lead, cols // 64).half())


def _mlp(hidden=2048, router=E, gate=True, shared=True, down=True):
    q8 = (torch.zeros(router, 512, dtype=torch.int32), torch.zeros(router, 32).half(), torch.zeros(router, 32).half())
    s = (_q(I, hidden), _q(I, hidden), _q(hidden, I)) if shared else (None,) * 3
    if not down:
        s = (*s[:2], None)
    return {"norm_w": torch.ones(hidden), "router": q8, "gate": tuple(t[:1] for t in q8) if gate else None,
            "experts": ExpertWeights(_q(I, hidden, E), _q(I, hidden, E), _q(hidden, I, E) if down else None, *s)}


def _stack(mlp=None, head=None):
    ctx = types.SimpleNamespace(device=0, handle=None, cfg=types.SimpleNamespace(max_batch=4, max_ctx=64, max_prefill_tokens=8))
    return AttentionStack(ctx, [{"mlp": mlp}], 2, 64, device="cpu", head=head)


@pytest.mark.parametrize("kw", [{"hidden": 1024}, {"router": 16}, {"shared": False}, {"down": False}])
def test_a_block_that_does_not_fit_is_refused_at_once(kw):
    with pytest.raises(ValueError):
        _stack(_mlp(**kw))


def test_blocks_that_fit():
    _stack(_mlp())
    _stack(_mlp(shared=False, gate=False))
    _stack(_mlp(gate=False))
    _stack(None)


def test_next_tokens_refusals():
    with pytest.raises(ValueError, match="without a head"):
        _stack().next_tokens(torch.zeros(1, 2048), torch.zeros(1))
    st = _stack(head={"norm_w": torch.ones(2048), "lm_head": _q(128, 2048)})
    for x in (torch.zeros(3, 2048), torch.zeros(0, 2048), torch.zeros(2, 1024), torch.zeros(2, 2048).bfloat16(), torch.zeros(2048)):
        with pytest.raises(ValueError, match="x must be"):
            st.next_tokens(x, torch.zeros(x.shape[0]))
