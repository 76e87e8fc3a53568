"""torch-facing wrappers over the C ABI.

Each wrapper mirrors one encoder block of the reference's per-layer schedule
(QwenQ4ActiveExpertStreamingRunner.swift:972-1167): it checks the tensors it
is handed, passes their device pointers and torch's current stream to the
library, and raises QffError on any non-zero status. Outputs are allocated
here only when the caller does not pass them.
"""
from __future__ import annotations

import ctypes
import operator
import struct

import torch

from ._lib import (BF16, F16, F32, Q4_MAX_PARTS, CtxCfg, DeltaNetParams, GqaParams, KvPages, MoeWeights, Q4Matrices,
                   Q4Part, QffError, check, lib)

_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
_f32, _bf16, _f16, _i32 = torch.float32, torch.bfloat16, torch.float16, torch.int32

# A decode-sized call is bound by the host: 12-17 us per call with a ctypes
# structure, c_void_p objects and torch's stream object built each time, 6-13
# of them Python (2-4 now). Addresses travel as plain ints, parameter blocks
# as packed bytes of the C layout (checked against the ctypes structures
# below), through function objects of their own whose block arguments are
# untyped pointers.
_P_DN = struct.Struct("PPPPf4x")
_P_GQA = struct.Struct("PPfiffi4x")
_P_KV = struct.Struct("PPPiii4x")
_P_Q4 = [struct.Struct("PPPi4xPi4xP" * n) for n in range(Q4_MAX_PARTS + 1)]
_P_Q4M = struct.Struct("PPP")
_P_MOE = struct.Struct("18P4i")
assert _P_Q4M.size == ctypes.sizeof(Q4Matrices) and _P_MOE.size == ctypes.sizeof(MoeWeights)
assert _P_DN.size == ctypes.sizeof(DeltaNetParams) and _P_GQA.size == ctypes.sizeof(GqaParams)
assert _P_Q4[1].size == ctypes.sizeof(Q4Part) and _P_KV.size == ctypes.sizeof(KvPages)


def _pack(layout: struct.Struct, pointers, *fields) -> bytes:
    try:
        return layout.pack(*pointers, *fields)
    except (struct.error, OverflowError):
        # as a ctypes structure takes them: a finite double past fp32 becomes
        # inf (for the library to judge), what is no number is a TypeError
        return layout.pack(*pointers, *(f if isinstance(f, int) else ctypes.c_float(f).value for f in fields))


_BLOCKS = (ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(DeltaNetParams), ctypes.POINTER(GqaParams), ctypes.POINTER(Q4Part), ctypes.POINTER(KvPages),
           ctypes.POINTER(Q4Matrices), ctypes.POINTER(MoeWeights))


class _Calls:
    """The hot entry points of the loaded library as functions of their own."""

    def __init__(self, L):
        for name in ("qff_q4_matmul", "qff_q4_matmul_parts", "qff_q4_norm_matmul_parts", "qff_router_top8",
                     "qff_deltanet_decode", "qff_deltanet_prefill", "qff_gqa_decode", "qff_gqa_prefill",
                     "qff_gqa_decode_paged", "qff_gqa_decode_shared", "qff_gqa_prefill_paged", "qff_pages_copy",
                     "qff_rms_norm", "qff_moe_gate_up", "qff_moe_down", "qff_sample"):
            fn = L[name]   # a new function object: the typed one of lib() stays as it is
            fn.argtypes = [ctypes.c_void_p if t in _BLOCKS else t for t in getattr(L, name).argtypes]
            fn.restype = ctypes.c_int
            setattr(self, name, fn)


_calls = None


def _hot() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls(lib())
    return _calls


def _code(t: torch.Tensor) -> int:
    c = _DT.get(t.dtype)
    if c is None:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return c


def _ptr(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError("tensor must live on the GPU")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return t.data_ptr()


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice

    def _stream() -> int:
        return _raw_stream(_device())
else:
    _raw_stream = None

    def _stream() -> int:
        return torch.cuda.current_stream().cuda_stream


def _rows(x: torch.Tensor, cols: int) -> torch.Tensor:
    """x as [batch, cols]."""
    return x if x.dim() == 2 and x.shape[1] == cols else x.reshape(-1, cols)


class Context:
    """Owns a qff_ctx: the device workspace for the hot calls (replaces the
    reference's MetalContext + Attention scratch set-up)."""

    def __init__(self, device: int = 0, max_batch: int = 32, max_ctx: int = 65536,
                 max_prefill_tokens: int = 8192):
        self.device = device
        h = ctypes.c_void_p()
        # (zeros stand for the defaults, as in the library; cfg holds what applies)
        cfg = CtxCfg(max_batch or 32, max_ctx or 65536, max_prefill_tokens or 8192)
        check("qff_ctx_create", lib().qff_ctx_create(ctypes.byref(h), device, ctypes.byref(cfg)))
        self.handle = h
        self.cfg = cfg

    def close(self):
        if self.handle:
            check("qff_ctx_destroy", lib().qff_ctx_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def q4_dequant(ctx: Context, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """w int32/uint32 [rows, cols/8]; scales/biases f16/bf16 [rows, cols/64] -> f32 [rows, cols]."""
    rows, c8 = w.shape
    if out is None:
        out = torch.empty(rows, c8 * 8, dtype=torch.float32, device=w.device)
    check("qff_q4_dequant", lib().qff_q4_dequant(ctx.handle, _stream(), _ptr(w), _ptr(scales),
                                                 _ptr(biases), _code(scales), _ptr(out), rows, c8 * 8))
    return out


def q4_matmul(ctx: Context, w, scales, biases, x: torch.Tensor, out=None,
              out_dtype=torch.float32) -> torch.Tensor:
    """x [batch, cols] (f32/bf16) -> y [batch, rows]."""
    rows, c8 = w.shape
    cols = c8 * 8
    x2 = _rows(x, cols)
    batch = x2.shape[0]
    if out is None:
        out = torch.empty(batch, rows, dtype=out_dtype, device=x.device)
    st = _hot().qff_q4_matmul(ctx.handle, _stream(), _ptr(w), _ptr(scales), _ptr(biases), _code(scales), _ptr(x2),
                              _code(x2), _ptr(out), _code(out), rows, cols, batch)
    if st:
        raise QffError("qff_q4_matmul", st)
    return out


def _q4_parts(parts, x, outs, out_dtypes, residuals):
    n = len(parts)
    if not 1 <= n <= Q4_MAX_PARTS:
        raise ValueError(f"1 .. {Q4_MAX_PARTS} parts")
    cols = parts[0][0].shape[1] * 8
    x2 = _rows(x, cols)
    batch = x2.shape[0]
    sdt = parts[0][1].dtype
    flat = []
    res = []
    for i, (w, s, b) in enumerate(parts):
        rows, c8 = w.shape[0], w.shape[1]
        if c8 * 8 != cols or s.dtype != sdt:
            raise ValueError("parts must share cols and scale dtype")
        if outs is not None:
            out = outs[i]
        else:
            dt = out_dtypes[i] if out_dtypes is not None else _f32
            out = torch.empty(batch, rows, dtype=dt, device=x.device)
        r = residuals[i] if residuals is not None else None
        if r is not None and (r.dtype != out.dtype or r.numel() != out.numel()):
            raise ValueError("a residual must match its output's dtype and size")
        flat += (_ptr(w), _ptr(s), _ptr(b), rows, _ptr(out), _code(out), _ptr(r) if r is not None else 0)
        res.append(out)
    return _P_Q4[n].pack(*flat), res, x2, cols, batch


def q4_matmul_parts(ctx: Context, parts, x: torch.Tensor, outs=None, out_dtypes=None, residuals=None):
    """One launch of y_p = x W_p^T (+ residual_p) for every part (w, scales,
    biases) in `parts` (all with the same cols and scale dtype), sharing x
    [batch, cols]. `residuals`: per part None or a tensor of the output's
    dtype and shape (may be the output itself). Returns the outputs
    [batch, rows_p]."""
    arr, res, x2, cols, batch = _q4_parts(parts, x, outs, out_dtypes, residuals)
    st = _hot().qff_q4_matmul_parts(ctx.handle, _stream(), arr, len(parts), _code(parts[0][1]), _ptr(x2), _code(x2),
                                    cols, batch)
    if st:
        raise QffError("qff_q4_matmul_parts", st)
    return res


def q4_norm_matmul_parts(ctx: Context, parts, x: torch.Tensor, norm_w: torch.Tensor, eps: float = 1e-6,
                         outs=None, out_dtypes=None, residuals=None):
    """The layer front-end: RMSNorm of each token of x (weight norm_w [cols],
    f32 or bf16, eps) feeding the grouped product of q4_matmul_parts."""
    arr, res, x2, cols, batch = _q4_parts(parts, x, outs, out_dtypes, residuals)
    if norm_w.numel() != cols:
        raise ValueError("norm_w must have cols entries")
    st = _hot().qff_q4_norm_matmul_parts(ctx.handle, _stream(), arr, len(parts), _code(parts[0][1]), _ptr(x2),
                                         _code(x2), _ptr(norm_w), _code(norm_w), eps, cols, batch)
    if st:
        raise QffError("qff_q4_norm_matmul_parts", st)
    return res


def q8_dequant(ctx: Context, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """w int32/uint32 [rows, cols/4]; scales/biases bf16/f16 [rows, cols/64] -> f32 [rows, cols]."""
    rows, c4 = w.shape
    if out is None:
        out = torch.empty(rows, c4 * 4, dtype=torch.float32, device=w.device)
    check("qff_q8_dequant", lib().qff_q8_dequant(ctx.handle, _stream(), _ptr(w), _ptr(scales),
                                                 _ptr(biases), _code(scales), _ptr(out), rows, c4 * 4))
    return out


def router_top8(ctx: Context, w, scales, biases, x: torch.Tensor, logits=None, indices=None, scores=None):
    """MoE router: Q8 logits of x [batch, cols] over the experts (rows of
    w), then the top eight per token. Returns (indices int32 [batch, 8],
    scores f32 [batch, 8], logits f32 [batch, experts])."""
    experts, c4 = w.shape
    cols = c4 * 4
    x2 = _rows(x, cols)
    batch = x2.shape[0]
    if logits is None:
        logits = torch.empty(batch, experts, dtype=_f32, device=x.device)
    if indices is None:
        indices = torch.empty(batch, 8, dtype=_i32, device=x.device)
    if scores is None:
        scores = torch.empty(batch, 8, dtype=_f32, device=x.device)
    st = _hot().qff_router_top8(ctx.handle, _stream(), _ptr(w), _ptr(scales), _ptr(biases), _code(scales), _ptr(x2),
                                _code(x2), _ptr(logits), _ptr(indices), _ptr(scores), experts, cols, batch)
    if st:
        raise QffError("qff_router_top8", st)
    return indices, scores, logits


def _require_f32(**tensors):
    for name, t in tensors.items():
        if t.dtype != _f32:
            raise TypeError(f"{name} must be float32")


def _dn_params(p: dict, eps: float) -> bytes:
    a_log, dt_bias, conv_w, norm_w = p["a_log"], p["dt_bias"], p["conv_w"], p["norm_w"]
    if a_log.dtype != _f32 or dt_bias.dtype != _f32 or conv_w.dtype != _f32 or norm_w.dtype != _f32:
        _require_f32(a_log=a_log, dt_bias=dt_bias, conv_w=conv_w, norm_w=norm_w)
    return _pack(_P_DN, (_ptr(a_log), _ptr(dt_bias), _ptr(conv_w), _ptr(norm_w)), eps)


def _check_dn_inputs(qkv, z, a, b, conv_state, ssm_state, n, seqs):
    """n tokens of `seqs` sequences: the shapes and element types the
    library assumes, checked before any pointer reaches it."""
    if z.dtype != qkv.dtype:
        raise TypeError("qkv and z must share a dtype")
    if a.dtype != _f32 or b.dtype != _f32 or conv_state.dtype != _f32 or ssm_state.dtype != _f32:
        _require_f32(a=a, b=b, conv_state=conv_state, ssm_state=ssm_state)
    if qkv.numel() != n * 8192 or z.numel() != n * 4096 or a.numel() != n * 32 or b.numel() != n * 32:
        raise ValueError("qkv, z, a, b must be [n, 8192], [n, 4096], [n, 32], [n, 32]")
    if conv_state.numel() != seqs * 8192 * 4 or ssm_state.numel() != seqs * 32 * 128 * 128:
        raise ValueError("conv_state / ssm_state must hold [8192, 4] / [32, 128, 128] per sequence")


def deltanet_decode(ctx: Context, params: dict, qkv, z, a, b, conv_state, ssm_state, out=None,
                    out_dtype=torch.bfloat16, eps: float = 1e-6) -> torch.Tensor:
    """One decode step for batch B. qkv [B,8192], z [B,4096] (same dtype), a, b
    [B,32] f32, conv_state [B,8192,4] f32, ssm_state [B,32,128,128] f32 (both
    updated in place) -> out [B,4096]."""
    B = qkv.shape[0]
    _check_dn_inputs(qkv, z, a, b, conv_state, ssm_state, B, B)
    if out is None:
        out = torch.empty(B, 4096, dtype=out_dtype, device=qkv.device)
    prm = _dn_params(params, eps)
    st = _hot().qff_deltanet_decode(ctx.handle, _stream(), prm, _ptr(qkv), _ptr(z), _code(qkv), _ptr(a), _ptr(b),
                                    _ptr(conv_state), _ptr(ssm_state), _ptr(out), _code(out), B)
    if st:
        raise QffError("qff_deltanet_decode", st)
    return out


def deltanet_prefill(ctx: Context, params: dict, qkv, z, a, b, conv_state, ssm_state, out=None,
                     out_dtype=torch.bfloat16, eps: float = 1e-6, chunk: int = 64) -> torch.Tensor:
    """T tokens of one sequence. qkv [T,8192], z [T,4096], a, b [T,32];
    conv_state [8192,4], ssm_state [32,128,128] updated in place -> out [T,4096]."""
    T = qkv.shape[0]
    _check_dn_inputs(qkv, z, a, b, conv_state, ssm_state, T, 1)
    if out is None:
        out = torch.empty(T, 4096, dtype=out_dtype, device=qkv.device)
    prm = _dn_params(params, eps)
    st = _hot().qff_deltanet_prefill(ctx.handle, _stream(), prm, _ptr(qkv), _ptr(z), _code(qkv), _ptr(a), _ptr(b),
                                     _ptr(conv_state), _ptr(ssm_state), _ptr(out), _code(out), T, chunk)
    if st:
        raise QffError("qff_deltanet_prefill", st)
    return out


def _check_gqa_inputs(q_gate, k, v, k_cache, v_cache, n):
    """The library reads q_gate, k and v with one element type and both
    caches as bf16 or both as fp16 (the reference's cache type): reject
    anything else before it reaches the device."""
    if (k_cache.dtype != _bf16 and k_cache.dtype != _f16) or v_cache.dtype != k_cache.dtype:
        raise TypeError("KV caches must both be bfloat16 or both float16")
    if k.dtype != q_gate.dtype or v.dtype != q_gate.dtype:
        raise TypeError("k and v must share q_gate's dtype")
    if q_gate.numel() != n * 16 * 512 or k.numel() != n * 512 or v.numel() != n * 512:
        raise ValueError("q_gate must be [n, 16, 512] and k, v [n, 2, 256]")


def _gqa_params(p: dict, theta, scale, eps, k_cache) -> bytes:
    return _pack(_P_GQA, (_ptr(p["q_norm_w"]), _ptr(p["k_norm_w"])), theta, 64, scale, eps, int(k_cache.dtype == _f16))


def gqa_decode(ctx: Context, params: dict, q_gate, k_new, v_new, k_cache, v_cache, positions,
               out=None, out_dtype=torch.bfloat16, theta=1e7, scale=1.0 / 16, eps=1e-6):
    """q_gate [B,16,512], k_new/v_new [B,2,256]; caches [B,max_ctx,2,256] bf16
    or fp16; positions int32 [B] (device) -> out [B,16,256]."""
    B = q_gate.shape[0]
    max_ctx = k_cache.shape[1]
    _check_gqa_inputs(q_gate, k_new, v_new, k_cache, v_cache, B)
    if k_cache.shape != (B, max_ctx, 2, 256) or v_cache.shape != k_cache.shape:
        raise ValueError("KV caches must be [B, max_ctx, 2, 256]")
    if positions.dtype != _i32 or positions.numel() != B:
        raise TypeError("positions must be int32 [B]")
    if out is None:
        out = torch.empty(B, 16, 256, dtype=out_dtype, device=q_gate.device)
    prm = _gqa_params(params, theta, scale, eps, k_cache)
    st = _hot().qff_gqa_decode(ctx.handle, _stream(), prm, _ptr(q_gate), _ptr(k_new), _ptr(v_new), _code(q_gate),
                               _ptr(k_cache), _ptr(v_cache), _ptr(positions), _ptr(out), _code(out), B, max_ctx)
    if st:
        raise QffError("qff_gqa_decode", st)
    return out


def gqa_prefill(ctx: Context, params: dict, q_gate, k, v, k_cache, v_cache, start_pos=0, out=None,
                out_dtype=torch.bfloat16, theta=1e7, scale=1.0 / 16, eps=1e-6):
    """q_gate [T,16,512], k/v [T,2,256]; caches [max_ctx,2,256] bf16 or fp16
    -> out [T,16,256]."""
    T = q_gate.shape[0]
    max_ctx = k_cache.shape[0]
    _check_gqa_inputs(q_gate, k, v, k_cache, v_cache, T)
    if k_cache.shape != (max_ctx, 2, 256) or v_cache.shape != k_cache.shape:
        raise ValueError("KV caches must be [max_ctx, 2, 256]")
    if out is None:
        out = torch.empty(T, 16, 256, dtype=out_dtype, device=q_gate.device)
    prm = _gqa_params(params, theta, scale, eps, k_cache)
    st = _hot().qff_gqa_prefill(ctx.handle, _stream(), prm, _ptr(q_gate), _ptr(k), _ptr(v), _code(q_gate),
                                _ptr(k_cache), _ptr(v_cache), start_pos, _ptr(out), _code(out), T, max_ctx)
    if st:
        raise QffError("qff_gqa_prefill", st)
    return out


def _ptr_on(ctx: Context, name: str, t: torch.Tensor, dtype=None) -> int:
    """The address of a contiguous tensor on the context's device."""
    if t.get_device() != ctx.device:
        raise ValueError(f"{name} must live on the context's device, cuda:{ctx.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    return t.data_ptr()


def _stream_of(ctx: Context) -> int:
    return torch.cuda.current_stream(ctx.device).cuda_stream if _raw_stream is None else _raw_stream(ctx.device)


def _paged_args(ctx: Context, params: dict, q_gate, k, v, k_pages, v_pages, table, rows, n, theta, scale, eps):
    """The checks and parameter blocks that the calls on a paged cache share:
    n tokens, `rows` rows of the table."""
    _check_gqa_inputs(q_gate, k, v, k_pages, v_pages, n)
    if k_pages.dim() != 4 or k_pages.shape[2:] != (2, 256) or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must be [num_pages, page_size, 2, 256]")
    if table.dim() != 2 or table.shape[0] != rows:
        raise ValueError(f"the page table must be [{rows}, entries]")
    qw, kw = params["q_norm_w"], params["k_norm_w"]
    if qw.numel() != 256 or kw.numel() != 256:
        raise ValueError("q_norm_w and k_norm_w must have 256 entries")
    prm = _pack(_P_GQA, (_ptr_on(ctx, "q_norm_w", qw, _f32), _ptr_on(ctx, "k_norm_w", kw, _f32)), theta, 64, scale, eps,
                int(k_pages.dtype == _f16))
    kv = _P_KV.pack(_ptr_on(ctx, "k_pages", k_pages), _ptr_on(ctx, "v_pages", v_pages),
                    _ptr_on(ctx, "the page table", table, _i32), k_pages.shape[0], k_pages.shape[1], table.shape[1])
    return prm, _ptr_on(ctx, "q_gate", q_gate), _ptr_on(ctx, "k", k), _ptr_on(ctx, "v", v), _code(q_gate), kv


def _paged_out(ctx: Context, q_gate, out, out_dtype, n):
    if out is None:
        out = torch.empty(n, 16, 256, dtype=out_dtype, device=q_gate.device)
    elif out.numel() != n * 4096:
        raise ValueError(f"out must be [{n}, 16, 256]")
    return out, _ptr_on(ctx, "out", out)


def gqa_decode_paged(ctx: Context, params: dict, q_gate, k_new, v_new, k_pages, v_pages, table, positions,
                     out=None, out_dtype=torch.bfloat16, theta=1e7, scale=1.0 / 16, eps=1e-6):
    """gqa_decode on a paged cache: k_pages / v_pages [num_pages, page_size, 2,
    256] bf16 or fp16, position p of sequence b at row p % page_size of page
    table[b, p // page_size] (table int32 [B, entries], on the device).
    q_gate [B,16,512], k_new / v_new [B,2,256], positions int32 [B] (device)
    -> out [B,16,256]; a position outside the table gives a NaN row."""
    B = q_gate.shape[0]
    prm, qp, kp, vp, code, kv = _paged_args(ctx, params, q_gate, k_new, v_new, k_pages, v_pages, table, B, B, theta,
                                            scale, eps)
    if positions.numel() != B:
        raise ValueError(f"positions must be [{B}]")
    out, op = _paged_out(ctx, q_gate, out, out_dtype, B)
    st = _hot().qff_gqa_decode_paged(ctx.handle, _stream_of(ctx), prm, qp, kp, vp, code, kv,
                                     _ptr_on(ctx, "positions", positions, _i32), op, _code(out), B)
    if st:
        raise QffError("qff_gqa_decode_paged", st)
    return out


def gqa_decode_shared(ctx: Context, params: dict, q_gate, k_new, v_new, k_pages, v_pages, table, positions, group,
                      shared_len, out=None, out_dtype=torch.bfloat16, theta=1e7, scale=1.0 / 16, eps=1e-6):
    """gqa_decode_paged where consecutive sequences with the same group >= 0
    hold the same K and V at their first positions (as many as the least of
    their shared_len), which are read once for up to 16 of them. group and
    shared_len: int32 [B] on the device; sequences of a negative group stand
    alone."""
    B = q_gate.shape[0]
    prm, qp, kp, vp, code, kv = _paged_args(ctx, params, q_gate, k_new, v_new, k_pages, v_pages, table, B, B, theta,
                                            scale, eps)
    if positions.numel() != B or group.numel() != B or shared_len.numel() != B:
        raise ValueError(f"positions, group and shared_len must be [{B}]")
    out, op = _paged_out(ctx, q_gate, out, out_dtype, B)
    st = _hot().qff_gqa_decode_shared(ctx.handle, _stream_of(ctx), prm, qp, kp, vp, code, kv,
                                      _ptr_on(ctx, "positions", positions, _i32), _ptr_on(ctx, "group", group, _i32),
                                      _ptr_on(ctx, "shared_len", shared_len, _i32), op, _code(out), B)
    if st:
        raise QffError("qff_gqa_decode_shared", st)
    return out


def gqa_prefill_paged(ctx: Context, params: dict, q_gate, k, v, k_pages, v_pages, table, start_pos=0, out=None,
                      out_dtype=torch.bfloat16, theta=1e7, scale=1.0 / 16, eps=1e-6):
    """gqa_prefill on a paged cache: T tokens of one sequence at positions
    start_pos .. start_pos + T - 1, appended to the pages its row of the table
    (int32 [entries]) names -> out [T,16,256]. Up to 42 tokens (fp32 outputs of a
    bf16 cache) or 64 (others) have gqa_decode_paged's precision, longer slices
    gqa_prefill's fp16 operands."""
    T = q_gate.shape[0]
    prm, qp, kp, vp, code, kv = _paged_args(ctx, params, q_gate, k, v, k_pages, v_pages,
                                            table[None] if table.dim() == 1 else table, 1, T, theta, scale, eps)
    out, op = _paged_out(ctx, q_gate, out, out_dtype, T)
    st = _hot().qff_gqa_prefill_paged(ctx.handle, _stream_of(ctx), prm, qp, kp, vp, code, kv, start_pos, op, _code(out),
                                      T)
    if st:
        raise QffError("qff_gqa_prefill_paged", st)
    return out


_nbytes = operator.attrgetter("nbytes")


def _host_i32(name, x) -> torch.Tensor:
    t = x if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=_i32)
    if t.is_cuda or t.dtype != _i32 or t.dim() != 1 or not t.is_contiguous():
        raise TypeError(f"{name} must be a list of ints or an int32 [n] tensor on the host")
    return t


def pages_copy(ctx: Context, pools, src, dst) -> None:
    """pool[dst[i]] = pool[src[i]] for every pool and i, in place. pools:
    tensors [num_pages, ...] of one number of pages and bytes per page (a
    multiple of 16): K and V pools, or DeltaNet states with one page per
    sequence. src, dst: page numbers, as lists or int32 host tensors; a
    destination may be neither repeated nor a source."""
    n = len(pools)
    if not n:
        raise ValueError("at least one pool")
    s, d = _host_i32("src", src), _host_i32("dst", dst)
    if s.numel() != d.numel():
        raise ValueError("src and dst must have the same length")
    # (whole-list checks: one by one they take as long as the launch for a model's twenty pools)
    pages, size = pools[0].shape[0], pools[0].nbytes
    if set(map(_nbytes, pools)) != {size} or {p.shape[0] for p in pools} != {pages}:
        raise ValueError("pools must have the same number of pages and bytes per page")
    size //= max(pages, 1)
    if set(map(torch.Tensor.get_device, pools)) != {ctx.device} or not all(map(torch.Tensor.is_contiguous, pools)):
        for p in pools:
            _ptr_on(ctx, "a pool", p)   # (names what is wrong)
    arr = struct.pack(f"{n}P", *map(torch.Tensor.data_ptr, pools))
    st = _hot().qff_pages_copy(ctx.handle, _stream_of(ctx), arr, n, size, pages, s.data_ptr(), d.data_ptr(), s.numel())
    if st:
        raise QffError("qff_pages_copy", st)


# ---- the expert block and the next token ---------------------------------------

_data_ptr = torch.Tensor.data_ptr
_WORDS, _SB = (torch.int32, torch.uint32), (torch.bfloat16, torch.float16)


def _check_matrix(name: str, q, bits: int, shape=None):
    """Whether (w, scales, biases) of affine-quantized matrices have shapes and types that the library reads."""
    w, s, b = q
    *rows, words = w.shape
    cols = words * (32 // bits)
    if w.dtype not in _WORDS:
        raise TypeError(f"{name}: the words must be int32")
    if s.dtype != b.dtype or s.dtype not in _SB:
        raise TypeError(f"{name}: scales and biases must both be bfloat16 or both float16")
    groups = (*rows, cols // 64)
    if cols % 64 or s.shape != groups or b.shape != groups:
        raise ValueError(f"{name}: scales and biases must be [.., cols / 64] of [.., {cols}]")
    if shape is not None and (*rows, cols) != shape:
        raise ValueError(f"{name} must be {list(shape)}")


def _matrix(ctx: Context, name: str, q, bits: int, shape=None):
    """Their addresses on the context's device, once they are."""
    _check_matrix(name, q, bits, shape)
    w, s, b = q
    return _ptr_on(ctx, name, w), _ptr_on(ctx, name + "'s scales", s), _ptr_on(ctx, name + "'s biases", b)


class ExpertWeights:
    """A layer's expert weights, each as (words, scales, biases) of affine-Q4
    matrices: gate, up [experts, inter, hidden], down [experts, hidden, inter] and
    the shared expert's [inter, hidden], [hidden, inter] (None: there is none).
    moe_gate_up needs gate and up, moe_down needs down; what only the other needs
    may be None. The tensors are kept; a call whose matrices no longer lie where they
    lay (set_, resize_, .data) checks all of them again and reads the new ones (the
    memory of the former is held until then)."""

    def __init__(self, gate=None, up=None, down=None, shared_gate=None, shared_up=None, shared_down=None):
        self.matrices = (gate, up, down, shared_gate, shared_up, shared_down)
        if gate is None and down is None:
            raise ValueError("either gate and up or down")
        if (gate is None) != (up is None) or (shared_gate is None) != (shared_up is None):
            raise ValueError("gate and up come together")
        if shared_gate is not None and gate is None or shared_down is not None and down is None:
            raise ValueError("a shared expert's matrices stand beside the routed experts'")
        if gate is not None and down is not None and (shared_gate is None) != (shared_down is None):
            raise ValueError("a shared expert has all three matrices")
        w = (gate if gate is not None else down)[0]
        if w.dim() != 3:
            raise ValueError("the experts' words must be [experts, rows, cols / 8]")
        rows, cols = w.shape[1], w.shape[2] * 8
        self.experts = w.shape[0]
        self.inter, self.hidden = (rows, cols) if gate is not None else (cols, rows)
        self.dtype = next(q[1].dtype for q in self.matrices if q is not None)
        # the tensors that gate_up and down read
        self._read = tuple(tuple(t for i in at for t in self.matrices[i] or ()) for at in ((0, 1, 3, 4), (2, 5)))
        # (context's device, both halves' addresses, parameter block, aliases): made by the first call, checked there. The
        # aliases keep the memory that was checked, so that nothing else can come to lie at its addresses.
        self._packed = None

    _NAMES = ("gate", "up", "down", "shared_gate", "shared_up", "shared_down")

    def check(self):
        """Raises where the matrices' shapes or types do not go together (as the first call does)."""
        up, down = (self.inter, self.hidden), (self.hidden, self.inter)
        for name, q, shape in zip(self._NAMES, self.matrices, [(self.experts, *s) for s in (up, up, down)] + [up, up, down]):
            if q is None:
                continue
            if q[1].dtype != self.dtype:
                raise TypeError("all scales and biases must have one type")
            _check_matrix(name, q, 4, shape)

    def _block(self, ctx: Context, half: int) -> bytes:
        """The parameter block for moe_gate_up (half 0) or moe_down (1)."""
        P = self._packed
        if P is not None and P[0] == ctx.device and P[1][half] == tuple(map(_data_ptr, self._read[half])):
            return P[2]
        self._packed = None
        self.check()
        flat = []
        for name, q in zip(self._NAMES, self.matrices):
            flat += _matrix(ctx, name, q, 4) if q is not None else (0, 0, 0)
        block = _P_MOE.pack(*flat, _DT[self.dtype], self.experts, self.hidden, self.inter)
        self._packed = (ctx.device, tuple(tuple(map(_data_ptr, r)) for r in self._read), block,
                        [t.detach() for r in self._read for t in r])
        return block


def _indices(ctx: Context, indices, tokens: int):
    """Their address and shape."""
    shape = indices.shape
    if len(shape) != 2 or shape[0] != tokens:
        raise ValueError(f"indices must be [{tokens}, top]")
    return _ptr_on(ctx, "indices", indices, _i32), shape


def rms_norm(ctx: Context, x: torch.Tensor, norm_w: torch.Tensor, eps: float = 1e-6, gate=None, out=None, out_dtype=None,
             coef=None):
    """RMSNorm of each row of x [tokens, cols] (f32 or bf16) with weight norm_w
    [cols] -> out (x's type unless out or out_dtype says otherwise; may be x). With
    `gate`, one affine-Q8 row (words [1, cols / 4], scales, biases [1, cols / 64]),
    (out, coef): coef [tokens] f32 = sigmoid(<gate, normed row>)."""
    if x.dim() != 2 or norm_w.numel() != x.shape[1]:
        raise ValueError("x must be [tokens, cols] and norm_w have cols entries")
    n, cols = x.shape
    if out is None:
        out = torch.empty(n, cols, dtype=out_dtype or x.dtype, device=x.device)
    elif out.shape != x.shape:
        raise ValueError(f"out must be [{n}, {cols}]")
    block, sb, cp = 0, BF16, 0
    if gate is not None:
        block, sb = _P_Q4M.pack(*_matrix(ctx, "gate", gate, 8, (1, cols))), _code(gate[1])
        if coef is None:
            coef = torch.empty(n, dtype=_f32, device=x.device)
        elif coef.numel() != n:
            raise ValueError(f"coef must be [{n}]")
        cp = _ptr_on(ctx, "coef", coef, _f32)
    st = _hot().qff_rms_norm(ctx.handle, _stream_of(ctx), _ptr_on(ctx, "x", x), _code(x), _ptr_on(ctx, "norm_w", norm_w),
                             _code(norm_w), eps, block, sb, _ptr_on(ctx, "out", out), _code(out), cp, cols, n)
    if st:
        raise QffError("qff_rms_norm", st)
    return out if gate is None else (out, coef)


def moe_gate_up(ctx: Context, experts: ExpertWeights, x: torch.Tensor, indices: torch.Tensor, out=None,
                out_dtype=torch.float32) -> torch.Tensor:
    """Every token through its experts' gate and up projections: x [tokens, hidden]
    (f32 or bf16), indices int32 [tokens, top] -> silu(x Wg^T) * (x Wu^T) [tokens,
    top (+ 1, the shared expert), inter] (f32, bf16 or f16). An index that is no
    expert's leaves its row as it was (a new tensor's: undefined)."""
    if experts.matrices[0] is None:
        raise ValueError("the weights have no gate and up matrices")
    shape = x.shape
    if len(shape) != 2 or shape[1] != experts.hidden:
        raise ValueError(f"x must be [tokens, {experts.hidden}]")
    n, block = shape[0], experts._block(ctx, 0)
    ip, (_, top) = _indices(ctx, indices, n)
    shape = (n, top + (experts.matrices[3] is not None), experts.inter)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=x.device)
    elif out.shape != shape:
        raise ValueError(f"out must be {list(shape)}")
    st = _hot().qff_moe_gate_up(ctx.handle, _stream_of(ctx), block, _ptr_on(ctx, "x", x), _code(x), ip, top,
                                _ptr_on(ctx, "out", out), _code(out), n)
    if st:
        raise QffError("qff_moe_gate_up", st)
    return out


def moe_down(ctx: Context, experts: ExpertWeights, h: torch.Tensor, indices: torch.Tensor, scores: torch.Tensor, coef=None,
             residual=None, out=None, out_dtype=torch.float32) -> torch.Tensor:
    """The experts' down projections of h [tokens, top (+ 1), inter] (f32, bf16 or
    f16), weighted with scores f32 [tokens, top] (the shared expert's row with coef f32
    [tokens], or 1) and summed on top of residual [tokens, hidden] (out's type; may be
    out) -> [tokens, hidden] (f32 or bf16)."""
    if experts.matrices[2] is None:
        raise ValueError("the weights have no down matrices")
    shape = h.shape
    n, block = shape[0], experts._block(ctx, 1)
    ip, (_, top) = _indices(ctx, indices, n)
    slots = top + (experts.matrices[5] is not None)
    if shape != (n, slots, experts.inter):
        raise ValueError(f"h must be [{n}, {slots}, {experts.inter}]")
    if scores.shape != (n, top):
        raise ValueError(f"scores must be {[n, top]}")
    shape = (n, experts.hidden)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=h.device)
    elif out.shape != shape:
        raise ValueError(f"out must be {list(shape)}")
    cp = rp = 0
    if coef is not None:
        if coef.numel() != n:
            raise ValueError(f"coef must be [{n}]")
        cp = _ptr_on(ctx, "coef", coef, _f32)
    if residual is not None:
        if residual.dtype != out.dtype or residual.shape != shape:
            raise ValueError("a residual must match its output's dtype and shape")
        rp = _ptr_on(ctx, "residual", residual)
    st = _hot().qff_moe_down(ctx.handle, _stream_of(ctx), block, _ptr_on(ctx, "h", h), _code(h), ip,
                             _ptr_on(ctx, "scores", scores, _f32), top, cp, rp, _ptr_on(ctx, "out", out),
                             _code(out), n)
    if st:
        raise QffError("qff_moe_down", st)
    return out


def _per_row(ctx: Context, name: str, t, n: int, dtype) -> int:
    if t is None:
        return 0
    if t.numel() != n:
        raise ValueError(f"{name} must be [{n}]")
    return _ptr_on(ctx, name, t, dtype)


def sample(ctx: Context, logits: torch.Tensor, u: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None,
           out=None, prob=None):
    """The next token of each sequence: logits [batch, vocab] (f32 or bf16), u f32
    [batch] in [0, 1) the random numbers; temperature, top_p, min_p f32 [batch] and
    top_k int32 [batch] on the device, or None (1, 1, 0 and 0, which filter
    nothing). Returns (tokens int32 [batch], what the drawn one had as its chance,
    f32 [batch]). temperature 0 takes the largest logit."""
    if logits.dim() != 2:
        raise ValueError("logits must be [batch, vocab]")
    n, vocab = logits.shape
    if out is None:
        out = torch.empty(n, dtype=_i32, device=logits.device)
    if prob is None:
        prob = torch.empty(n, dtype=_f32, device=logits.device)
    if u is None:
        raise TypeError("u must be float32 random numbers")
    st = _hot().qff_sample(ctx.handle, _stream_of(ctx), _ptr_on(ctx, "logits", logits), _code(logits),
                           _per_row(ctx, "u", u, n, _f32), _per_row(ctx, "temperature", temperature, n, _f32),
                           _per_row(ctx, "top_k", top_k, n, _i32), _per_row(ctx, "top_p", top_p, n, _f32),
                           _per_row(ctx, "min_p", min_p, n, _f32), _per_row(ctx, "out", out, n, _i32),
                           _per_row(ctx, "prob", prob, n, _f32), vocab, n)
    if st:
        raise QffError("qff_sample", st)
    return out, prob


__all__ = ["Context", "QffError", "q4_dequant", "q4_matmul", "deltanet_decode", "deltanet_prefill",
           "gqa_decode", "gqa_prefill", "gqa_decode_paged", "gqa_decode_shared", "gqa_prefill_paged", "pages_copy",
           "ExpertWeights", "rms_norm", "moe_gate_up", "moe_down", "sample", "BF16", "F16", "F32"]
