"""The decoder stack: the per-layer schedule of
QwenQ4ActiveExpertStreamingRunner.forwardToken (Runner:924-1167) over the C
ABI. A layer whose dict has no "mlp" has identity in the expert block's place.

Layer l is full attention when l % 4 == 3, Gated DeltaNet otherwise
(Runner:554-556). Each layer reads the residual stream x [B, 2048] and adds
its attention output back into it (Runner:1034-1040, 1162-1166):

  DeltaNet   input RMSNorm + fused in-projection qkv|z|b|a (Runner:973-997)
             -> conv1d + gated delta rule + gated RMSNorm (Runner:1001-1022)
             -> out_proj, added into x (Runner:1024-1040)
  full attn  input RMSNorm + q|gate, k, v projections (Runner:1043-1074)
             -> split / head norms / RoPE / KV append / attention / gate
                (Runner:1076-1150) -> o_proj, added into x (Runner:1152-1166)
  "mlp"      post-attention RMSNorm and the shared expert's coefficient ->
             router -> the experts' gate and up -> down, weighted and added into x

and from the last layer's x, final RMSNorm + head product -> the next tokens
(next_tokens), for a stack that was given its head.

The residual stream and every intermediate are fp32, as the reference keeps
them (hiddenBuf0/1, qkvOutBuf, ... are float buffers, Runner:346-401); the KV
caches are bf16, one flat cache per sequence or, with a PageTable, pages of one
pool per layer, which sequences that share a prefix hold together. Layers take the tensors Checkpoint.deltanet_layer /
gqa_layer return, so a stack can come from a checkpoint or from synthetic
weights of the same layout.
"""
from __future__ import annotations

import torch

from . import ops
from .pages import OutOfPages

HIDDEN = 2048
MOST_VOCAB, MOST_INTER = 262144, 4096   # of the sampling and the expert block
ROUTER_EXPERTS = range(8, 257)


def is_full_attention(l: int) -> bool:
    return l % 4 == 3


class AttentionStack:
    """Layers, their per-sequence state and the scratch tensors of one decode
    step for `batch` sequences. `layers[l]` is a dict with the keys of
    Checkpoint.deltanet_layer (DeltaNet) or Checkpoint.gqa_layer (full
    attention); the kind follows l % 4 == 3 unless `kinds` says otherwise. Its
    "mlp" is what Checkpoint.expert_layer returns; `head` what Checkpoint.head
    returns (None: the stack ends with x).
    States: DeltaNet conv [B, 8192, 4] / ssm [B, 32, 128, 128] fp32, full
    attention K / V caches [B, max_ctx, 2, 256] bf16; pass them in `states`
    or get zero states.

    With `pages` (a PageTable of `batch` slots), full attention keeps k_pages /
    v_pages [num_pages, page_size, 2, 256] instead, slot b of the table is
    sequence b, and sequences can be filled a prompt slice at a time (prefill),
    forked, released and compacted. Before each decode step, captured or not,
    reserve() gives the new tokens their places."""

    def __init__(self, ctx: ops.Context, layers, batch: int, max_ctx: int, states=None, kinds=None,
                 eps: float = 1e-6, device="cuda", pages=None, head=None):
        self.ctx = ctx
        self.layers = list(layers)
        self.B = batch
        self.max_ctx = max_ctx
        self.eps = eps
        self.pages = pages
        if pages is not None:
            # (here, and not by the first call that finds out with its positions reserved)
            if len(pages.lengths) != batch or batch > ctx.cfg.max_batch:
                raise ValueError(f"the page table must have {batch} slots, and the context's max_batch as many")
            if pages.cols > -(-ctx.cfg.max_ctx // pages.page_size):
                raise ValueError(f"the page table's rows of {pages.cols * pages.page_size} positions exceed the context's "
                                 f"max_ctx of {ctx.cfg.max_ctx}")
        self._parked = {}   # slot -> its recurrent states, while it sits out decode steps
        self.kinds = list(kinds) if kinds is not None else \
            ["gqa" if is_full_attention(l) else "dn" for l in range(len(self.layers))]
        if states is None:
            states = []
            for kind in self.kinds:
                if kind == "dn":
                    states.append({"conv_state": torch.zeros(batch, 8192, 4, device=device),
                                   "ssm_state": torch.zeros(batch, 32, 128, 128, device=device)})
                elif pages is not None:
                    shape = (len(pages.refs), pages.page_size, 2, 256)
                    states.append({k: torch.zeros(shape, dtype=torch.bfloat16, device=device)
                                   for k in ("k_pages", "v_pages")})
                else:
                    states.append({"k_cache": torch.zeros(batch, max_ctx, 2, 256, dtype=torch.bfloat16,
                                                          device=device),
                                   "v_cache": torch.zeros(batch, max_ctx, 2, 256, dtype=torch.bfloat16,
                                                          device=device)})
        self.states = states
        f32 = dict(dtype=torch.float32, device=device)
        self.qkv = torch.empty(batch, 8192, **f32)
        self.z = torch.empty(batch, 4096, **f32)
        self.a = torch.empty(batch, 32, **f32)
        self.b = torch.empty(batch, 32, **f32)
        self.core = torch.empty(batch, 4096, **f32)
        self.qg = torch.empty(batch, 8192, **f32)
        self.kn = torch.empty(batch, 512, **f32)
        self.vn = torch.empty(batch, 512, **f32)
        self.att = torch.empty(batch, 16, 256, **f32)
        self._block = {}   # an expert block's tensors by what its shapes depend on: layers of one shape share them
        for L in self.layers:
            M = L.get("mlp")
            if M is None:
                continue
            self._check_block(M)
            if self._shape(M) not in self._block:
                self._block[self._shape(M)] = self._block_tensors(M, batch, device)
        self._placed = not self._block   # whether _ready has seen the blocks' tensors
        self.head = head
        if (head is not None or self._block) and batch > ctx.cfg.max_batch:
            raise ValueError(f"a batch of {batch} exceeds the context's max_batch of {ctx.cfg.max_batch}")
        if head is not None:
            self._check_norm("the head's", head["norm_w"])
            vocab = head["lm_head"][0].shape[0]
            ops._check_matrix("lm_head", head["lm_head"], 4, (vocab, HIDDEN))
            if not 1 <= vocab <= MOST_VOCAB:
                raise ValueError(f"lm_head must have 1 .. {MOST_VOCAB} rows")
            self.logits = torch.empty(batch, head["lm_head"][0].shape[0], **f32)
            self.tokens = torch.empty(batch, dtype=torch.int32, device=device)
            self.chances = torch.empty(batch, **f32)

    @staticmethod
    def _check_norm(whose, w):
        if w.numel() != HIDDEN or w.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"{whose} norm_w must be float32 or bfloat16 [{HIDDEN}]")

    def _check_block(self, M):
        """What the calls of an expert block would refuse, whatever the device (here, and not by one of them with the
        layer's recurrent state or its cache advanced before it)."""
        E = M["experts"]
        if E.hidden != HIDDEN or None in (E.matrices[0], E.matrices[2]):
            raise ValueError(f"a layer's experts need gate, up and down of {HIDDEN} columns of x")
        if M["router"][0].shape[0] != E.experts:
            raise ValueError("a layer's router must have a row for each of its experts")
        if E.experts not in ROUTER_EXPERTS or E.inter > MOST_INTER:
            raise ValueError(f"a layer takes {ROUTER_EXPERTS.start} .. {ROUTER_EXPERTS.stop - 1} experts of up to {MOST_INTER} rows")
        if M["gate"] is not None and E.matrices[3] is None:
            raise ValueError("a shared expert's gate needs a shared expert")
        self._check_norm("a layer's", M["norm_w"])
        ops._check_matrix("router", M["router"], 8, (E.experts, HIDDEN))
        if M["gate"] is not None:
            ops._check_matrix("gate", M["gate"], 8, (1, HIDDEN))
        E.check()

    def _ready(self):
        """The rest of it, once, ahead of the first step or slice: where the blocks' tensors lie, by calls of no tokens."""
        if self._placed:
            return
        ctx = self.ctx
        for L in self.layers:
            M = L.get("mlp")
            if M is None:
                continue
            x, idx, sc = self._none(M["norm_w"].device)
            ops.rms_norm(ctx, x, M["norm_w"], self.eps, gate=M["gate"])
            ops._matrix(ctx, "router", M["router"], 8)
            h = ops.moe_gate_up(ctx, M["experts"], x, idx)
            ops.moe_down(ctx, M["experts"], h, idx, sc)
        self._placed = True

    @staticmethod
    def _none(device):
        """x, indices and scores of no tokens."""
        return (torch.empty(0, HIDDEN, device=device), torch.empty(0, 8, dtype=torch.int32, device=device),
                torch.empty(0, 8, device=device))

    @staticmethod
    def _shape(M):
        E = M["experts"]
        return E.experts, E.inter, E.matrices[3] is not None

    @staticmethod
    def _block_tensors(M, n, device):
        E = M["experts"]
        f32 = dict(dtype=torch.float32, device=device)
        return (torch.empty(n, HIDDEN, **f32), torch.empty(n, **f32), torch.empty(n, E.experts, **f32),
                torch.empty(n, 8, dtype=torch.int32, device=device), torch.empty(n, 8, **f32),
                torch.empty(n, 8 + (E.matrices[3] is not None), E.inter, **f32))

    def _experts(self, M, x: torch.Tensor, tensors):
        """A layer's expert block on the residual stream, in place."""
        xn, coef, logits, indices, scores, h = tensors
        if M["gate"] is not None:
            ops.rms_norm(self.ctx, x, M["norm_w"], self.eps, gate=M["gate"], out=xn, coef=coef)
        else:
            ops.rms_norm(self.ctx, x, M["norm_w"], self.eps, out=xn)
        ops.router_top8(self.ctx, *M["router"], xn, logits=logits, indices=indices, scores=scores)
        ops.moe_gate_up(self.ctx, M["experts"], xn, indices, out=h)
        ops.moe_down(self.ctx, M["experts"], h, indices, scores, coef=coef if M["gate"] is not None else None,
                     residual=x, out=x)

    def layer_step(self, l: int, x: torch.Tensor, positions: torch.Tensor):
        """Layer l of one decode step: x [B, 2048] fp32, updated in place."""
        L, S, B = self.layers[l], self.states[l], self.B
        ctx, eps = self.ctx, self.eps
        if self.kinds[l] == "dn":
            ops.q4_norm_matmul_parts(ctx, L["in_proj"], x, L["in_norm_w"], eps,
                                     outs=(self.qkv, self.z, self.b, self.a))
            ops.deltanet_decode(ctx, L["params"], self.qkv, self.z, self.a, self.b, S["conv_state"],
                                S["ssm_state"], out=self.core, eps=eps)
            ops.q4_matmul_parts(ctx, [L["out_proj"]], self.core, outs=(x,), residuals=(x,))
        else:
            ops.q4_norm_matmul_parts(ctx, L["in_proj"], x, L["in_norm_w"], eps,
                                     outs=(self.qg, self.kn, self.vn))
            new = (self.qg.view(B, 16, 512), self.kn.view(B, 2, 256), self.vn.view(B, 2, 256))
            if self.pages is None:
                ops.gqa_decode(ctx, L["params"], *new, S["k_cache"], S["v_cache"], positions, out=self.att,
                               eps=eps)
            else:
                P = self.pages
                ops.gqa_decode_shared(ctx, L["params"], *new, S["k_pages"], S["v_pages"], P.table, positions,
                                      P.group, P.shared_len, out=self.att, eps=eps)
            ops.q4_matmul_parts(ctx, [L["out_proj"]], self.att.view(B, 4096), outs=(x,), residuals=(x,))
        M = L.get("mlp")
        if M is not None:
            self._experts(M, x, self._block[self._shape(M)])

    def next_tokens(self, x: torch.Tensor, u: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None):
        """The next tokens from the last layer's rows x [n, 2048] fp32, n <= batch (a
        decode step's, or a prompt's last row), with the random numbers and
        settings of ops.sample. Returns (tokens int32 [n], their chances f32 [n]),
        views of the stack's own tensors that the next call writes again."""
        if self.head is None:
            raise ValueError("the stack was made without a head")
        n = x.shape[0]
        if x.dtype != torch.float32 or x.dim() != 2 or x.shape[1] != HIDDEN or not 1 <= n <= self.B:
            raise ValueError(f"x must be float32 [1 .. {self.B}, {HIDDEN}]")
        logits = self.logits[:n]
        ops.q4_norm_matmul_parts(self.ctx, [self.head["lm_head"]], x, self.head["norm_w"], self.eps, outs=(logits,))
        return ops.sample(self.ctx, logits, u, temperature, top_k, top_p, min_p, out=self.tokens[:n], prob=self.chances[:n])

    def decode_step(self, x: torch.Tensor, positions: torch.Tensor):
        """Every layer in order: x [B, 2048] fp32 (the residual stream, in
        place), positions int32 [B] on the device (the new token's position
        in each sequence; full-attention layers append there)."""
        if x.dtype != torch.float32 or tuple(x.shape) != (self.B, HIDDEN):
            raise ValueError(f"x must be float32 [{self.B}, {HIDDEN}]")
        # (here, and not by the first full-attention layer, with recurrent states advanced before it)
        if positions.dtype != torch.int32 or positions.numel() != self.B:
            raise TypeError(f"positions must be int32 [{self.B}]")
        if positions.device != x.device or not positions.is_contiguous():
            raise ValueError("positions must be contiguous, on x's device")
        self._ready()
        for l in range(len(self.layers)):
            self.layer_step(l, x, positions)

    # ---- sequences of a paged stack ------------------------------------------

    def _paged(self):
        if self.pages is None:
            raise ValueError("the stack was made without pages")
        return self.pages

    def _recurrent(self):
        return [S[k] for kind, S in zip(self.kinds, self.states) if kind == "dn" for k in ("conv_state", "ssm_state")]

    def _park(self, slot: int):
        """Keeps a slot's recurrent states aside: a decode step advances those of
        every slot, and a slot without a position has no input."""
        if slot not in self._parked:
            self._parked[slot] = [t[slot].clone() for t in self._recurrent()]

    def _unpark(self, slot: int):
        for t, kept in zip(self._recurrent(), self._parked.pop(slot, [])):
            t[slot].copy_(kept)

    def _copy_pages(self, src, dst):
        pools = [S[k] for kind, S in zip(self.kinds, self.states) if kind == "gqa" for k in ("k_pages", "v_pages")]
        if src and pools:
            ops.pages_copy(self.ctx, pools, src, dst)

    def reserve(self, positions):
        """Places for one decode step's tokens: positions[b] is the new token's
        position in slot b, negative for a slot that takes no part (what it holds
        stays as it is, for a later step or slice). Each follows those that the slot
        holds (it may lie among them in a stack without recurrent layers, whose
        states cannot go back). Pages that a slot shares and is about to write are
        copied; an empty slot's position 0 begins a sequence (zero recurrent
        states). Where the pool runs out (OutOfPages), no slot holds a position more
        than before; the copies made for the slots before that one stay theirs."""
        pages, copies = self._paged(), []
        if len(positions) != self.B:
            raise ValueError(f"positions must have {self.B} entries")
        self._ready()
        held = list(pages.lengths)
        for b, p in enumerate(positions):
            if p > held[b] or 0 <= p < held[b] and "dn" in self.kinds:
                raise ValueError(f"slot {b} holds {held[b]} positions: position {p} does not follow them")
            if p >= pages.cols * pages.page_size:
                raise ValueError(f"slot {b}: position {p} does not fit {pages.cols} pages")
        try:
            for b, p in enumerate(positions):
                if p < 0:
                    if pages.lengths[b]:
                        self._park(b)
                    continue
                empty = not pages.lengths[b]
                copies += pages.reserve(b, p, p + 1)
                if empty:
                    for t in self._recurrent():
                        t[b].zero_()
                self._unpark(b)
        except OutOfPages:
            for b, n in enumerate(held):
                pages.truncate(b, n)
            raise
        finally:
            self._copy_pages([s for s, _ in copies], [d for _, d in copies])
            self.pages.sync()

    def prefill(self, slot: int, x: torch.Tensor, start: int = 0):
        """A prompt slice of T tokens of one slot through every layer: x [T, 2048]
        fp32 (the residual stream, in place) at positions start .. start + T - 1,
        behind those that the slot holds; start 0 begins a sequence in an empty slot
        (zero recurrent states). A refused call changes nothing."""
        if x.dtype != torch.float32 or x.dim() != 2 or x.shape[1] != HIDDEN:
            raise ValueError(f"x must be float32 [T, {HIDDEN}]")
        if x.get_device() != self.ctx.device or not x.is_contiguous():
            raise ValueError(f"x must be contiguous, on the context's device, cuda:{self.ctx.device}")
        P, T, ctx, eps = self._paged(), x.shape[0], self.ctx, self.eps
        P.check_slot(slot)
        if T > ctx.cfg.max_prefill_tokens or start + T > ctx.cfg.max_ctx:
            raise ValueError(f"{T} tokens from {start}: the context takes slices of {ctx.cfg.max_prefill_tokens} up to "
                             f"position {ctx.cfg.max_ctx}")
        if start != P.lengths[slot] and "dn" in self.kinds:
            raise ValueError(f"slot {slot} holds {P.lengths[slot]} positions: a slice follows them, or begins in a released slot")
        self._ready()
        copies = P.reserve(slot, start, start + T)
        self._unpark(slot)
        self._copy_pages([s for s, _ in copies], [d for _, d in copies])
        P.sync()
        blocks = {}
        for kind, L, S in zip(self.kinds, self.layers, self.states):
            y = ops.q4_norm_matmul_parts(ctx, L["in_proj"], x, L["in_norm_w"], eps)
            if kind == "dn":
                conv, ssm = S["conv_state"][slot], S["ssm_state"][slot]
                if start == 0:
                    conv.zero_()
                    ssm.zero_()
                core = ops.deltanet_prefill(ctx, L["params"], y[0], y[1], y[3], y[2], conv, ssm, out_dtype=torch.float32,
                                            eps=eps)
            else:
                core = ops.gqa_prefill_paged(ctx, L["params"], y[0].view(T, 16, 512), y[1].view(T, 2, 256),
                                             y[2].view(T, 2, 256), S["k_pages"], S["v_pages"], P.table[slot],
                                             start_pos=start, out_dtype=torch.float32, eps=eps).view(T, 4096)
            ops.q4_matmul_parts(ctx, [L["out_proj"]], core, outs=(x,), residuals=(x,))
            M = L.get("mlp")
            if M is not None:
                shape = self._shape(M)
                if shape not in blocks:
                    blocks[shape] = self._block_tensors(M, T, x.device)
                self._experts(M, x, blocks[shape])

    def fork(self, src: int, dsts):
        """Slots `dsts` (empty) go on from where slot src stands: its pages are
        held by all, its recurrent states copied. Neighbouring slots read what
        they share once."""
        dsts, pages = list(dsts), self._paged()
        for s in (src, *dsts):
            pages.check_slot(s)
        if src in dsts or len(set(dsts)) < len(dsts) or any(pages.lengths[d] for d in dsts):
            raise ValueError("a fork goes into empty slots")
        for d in dsts:
            pages.fork(src, d)
        self._unpark(src)
        recurrent = [S for kind, S in zip(self.kinds, self.states) if kind == "dn"]
        if dsts and recurrent:
            for k in ("conv_state", "ssm_state"):
                ops.pages_copy(self.ctx, [S[k] for S in recurrent], [src] * len(dsts), dsts)
        self.pages.sync()

    def release(self, slot: int):
        """Ends a slot's sequence; pages that no other slot holds are free again."""
        self._paged().release(slot)
        self._parked.pop(slot, None)
        self.pages.sync()

    def compact(self) -> int:
        """Moves the pages in use to the front of every pool; returns their
        number."""
        self._copy_pages(*self._paged().compact())
        self.pages.sync()
        return int((self.pages.refs > 0).sum())


def random_q4(rows: int, cols: int, gen: torch.Generator, device="cuda"):
    """An affine-Q4 weight with uniform nibbles, fp16 scales U(0.005, 0.02)
    and fp16 biases N(0, 0.05) (the config-3/4 distributions), made on the
    device."""
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, cols // 8), dtype=torch.int32, device=device,
                      generator=gen)
    sc = (torch.rand(rows, cols // 64, device=device, generator=gen) * 0.015 + 0.005).half()
    bi = (torch.randn(rows, cols // 64, device=device, generator=gen) * 0.05).half()
    return w, sc, bi


def random_q8(rows: int, cols: int, gen: torch.Generator, device="cuda"):
    """An affine-Q8 weight of about the same spread, fp16 scales and biases."""
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, cols // 4), dtype=torch.int32, device=device, generator=gen)
    sc = (torch.rand(rows, cols // 64, device=device, generator=gen) * 0.0009 + 0.0003).half()
    return w, sc, (-127.5 * sc.float()).half()


def random_mlp(experts: int, inter: int, gen: torch.Generator, device="cuda"):
    """An expert block with a shared expert, random weights (see random_q4),
    post-attention RMSNorm weights 1."""
    def stacked(rows, cols):
        w, sc, bi = random_q4(experts * rows, cols, gen, device)
        return w.view(experts, rows, -1), sc.view(experts, rows, -1), bi.view(experts, rows, -1)
    return {"norm_w": torch.ones(HIDDEN, device=device), "router": random_q8(experts, HIDDEN, gen, device),
            "gate": random_q8(1, HIDDEN, gen, device),
            "experts": ops.ExpertWeights(stacked(inter, HIDDEN), stacked(inter, HIDDEN), stacked(HIDDEN, inter),
                                         random_q4(inter, HIDDEN, gen, device), random_q4(inter, HIDDEN, gen, device),
                                         random_q4(HIDDEN, inter, gen, device))}


def random_layers(n: int, gen: torch.Generator, dn_params: dict, gqa_params: dict, device="cuda"):
    """n layers of the l % 4 == 3 pattern with random affine-Q4 projections
    and input-RMSNorm weights 1; the layer constants (A_log, dt_bias, conv
    and norm weights, q/k norm weights) are shared dicts of fp32 tensors."""
    ones = torch.ones(HIDDEN, device=device)
    layers = []
    for l in range(n):
        if is_full_attention(l):
            layers.append({"in_norm_w": ones,
                           "in_proj": [random_q4(r, HIDDEN, gen, device) for r in (8192, 512, 512)],
                           "out_proj": random_q4(HIDDEN, 4096, gen, device), "params": gqa_params})
        else:
            layers.append({"in_norm_w": ones,
                           "in_proj": [random_q4(r, HIDDEN, gen, device) for r in (8192, 4096, 32, 32)],
                           "out_proj": random_q4(HIDDEN, 4096, gen, device), "params": dn_params})
    return layers
