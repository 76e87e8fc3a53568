"""The paged-cache calls on the host, without a GPU: what the library refuses
(a C++ program over the C entry points, tests/host_checks/paged_checks.cpp)
and what the torch wrappers check before they reach it."""
import os
import subprocess
import types

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_refusals(tmp_path):
    import qff
    from qff._lib import LIB_PATH
    qff.lib()
    exe = str(tmp_path / "paged_checks")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-w", "-I" + os.path.join(rocm, "include"),
                        "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "qwen-fieldfare_amd", "csrc"),
                        os.path.join(ROOT, "tests", "host_checks", "paged_checks.cpp"), LIB_PATH,
                        "-L" + os.path.join(rocm, "lib"), "-lamdhip64", "-Wl,-rpath," + os.path.dirname(LIB_PATH),
                        "-Wl,-rpath," + os.path.join(rocm, "lib"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:]


def _args(B=2, kv=torch.bfloat16):
    p = {"q_norm_w": torch.ones(256), "k_norm_w": torch.ones(256)}
    return {"params": p, "q_gate": torch.zeros(B, 16, 512), "k_new": torch.zeros(B, 2, 256), "v_new": torch.zeros(B, 2, 256),
            "k_pages": torch.zeros(4, 16, 2, 256, dtype=kv), "v_pages": torch.zeros(4, 16, 2, 256, dtype=kv),
            "table": torch.zeros(B, 2, dtype=torch.int32), "positions": torch.zeros(B, dtype=torch.int32)}


@pytest.mark.parametrize("change,error", [
    ({}, ValueError),                                                     # host tensors: not on the context's device
    ({"k_pages": torch.zeros(4, 16, 2, 256)}, TypeError),
    ({"v_pages": torch.zeros(4, 16, 2, 256, dtype=torch.float16)}, TypeError),
    ({"k_new": torch.zeros(2, 2, 256, dtype=torch.bfloat16)}, TypeError),
    ({"v_pages": torch.zeros(5, 16, 2, 256, dtype=torch.bfloat16)}, ValueError),
    ({"k_pages": torch.zeros(4, 16, 256, 2, dtype=torch.bfloat16)}, ValueError),
    ({"q_gate": torch.zeros(2, 16, 511)}, ValueError),
    ({"k_new": torch.zeros(3, 2, 256)}, ValueError),
    ({"table": torch.zeros(3, 2, dtype=torch.int32)}, ValueError),
    ({"table": torch.zeros(2, dtype=torch.int32)}, ValueError),
    ({"params": {"q_norm_w": torch.ones(255), "k_norm_w": torch.ones(256)}}, ValueError)])
def test_wrapper_checks(change, error):
    from qff import ops
    ctx = types.SimpleNamespace(device=0, handle=None)
    a = {**_args(), **change}
    with pytest.raises(error):
        ops.gqa_decode_paged(ctx, **a)
    one = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(error):
        ops.gqa_decode_shared(ctx, **a, group=one, shared_len=one)
    if "table" not in change:
        a["k"], a["v"], a["table"] = a.pop("k_new"), a.pop("v_new"), a["table"][0]
        a.pop("positions")
        with pytest.raises(error):
            ops.gqa_prefill_paged(ctx, **a)


def test_copy_wrapper_checks():
    from qff import ops
    ctx = types.SimpleNamespace(device=0, handle=None)
    pool = torch.zeros(4, 16)
    for pools, src, dst, error in (([], [0], [1], ValueError), ([pool], [0, 1], [2], ValueError),
                                   ([pool, pool[:3]], [0], [1], ValueError), ([pool], [0], [1], ValueError),
                                   ([pool], torch.tensor([0]), torch.tensor([1]), TypeError),
                                   ([pool], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), TypeError)):
        with pytest.raises(error):
            ops.pages_copy(ctx, pools, src, dst)


def test_kv_pages_block_matches_the_structure():
    import ctypes

    from qff import ops
    from qff._lib import KvPages
    f = (0x1122334455667788, 0x1122334455667799, 0x11223344556677aa, 3, 64, 17)
    assert ops._P_KV.pack(*f) == bytes(KvPages(*f)) and ops._P_KV.size == ctypes.sizeof(KvPages)


class _Calls:
    """In the library's place: takes every call, and remembers their names."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        return lambda *args: self.made.append(name) or 0


@pytest.fixture
def on_host(monkeypatch):
    """(context, calls): host tensors lie on this context's device (-1), so that
    nothing but the check in question can refuse a call."""
    from qff import ops
    calls = _Calls()
    monkeypatch.setattr(ops, "_hot", lambda: calls)
    monkeypatch.setattr(ops, "_stream_of", lambda ctx: 0)
    return types.SimpleNamespace(device=-1, handle=None), calls


def _each_call(ops, ctx, a):
    """The decode, the shared decode and the prefill of these arguments."""
    B = a["positions"].numel()
    yield "qff_gqa_decode_paged", lambda: ops.gqa_decode_paged(ctx, **a)
    ints = torch.zeros(B, dtype=torch.int32)
    yield "qff_gqa_decode_shared", lambda: ops.gqa_decode_shared(ctx, **a, group=ints, shared_len=ints)
    one = {k: a[k] for k in ("params", "q_gate", "k_pages", "v_pages") if k in a} | {"k": a["k_new"], "v": a["v_new"], "table": a["table"][0]}
    yield "qff_gqa_prefill_paged", lambda: ops.gqa_prefill_paged(ctx, **one, **({"out": a["out"]} if "out" in a else {}))


def test_wrappers_pass_on_what_they_check(on_host):
    from qff import ops
    ctx, calls = on_host
    for kv in (torch.bfloat16, torch.float16):
        for name, call in _each_call(ops, ctx, _args(kv=kv)):
            assert call().shape == (2, 16, 256) and calls.made[-1] == name
    ops.pages_copy(ctx, [torch.zeros(4, 16)], [0], [1])
    assert calls.made[-1] == "qff_pages_copy"


_BF, _NORMS = torch.bfloat16, "q_norm_w and k_norm_w must have 256"


@pytest.mark.parametrize("change,error,match", [
    ({"k_pages": torch.zeros(4, 16, 2, 256)}, TypeError, "KV caches must both"),
    ({"v_pages": torch.zeros(4, 16, 2, 256, dtype=torch.float16)}, TypeError, "KV caches must both"),
    ({"k_new": torch.zeros(2, 2, 256, dtype=_BF)}, TypeError, "share q_gate's dtype"),
    ({"v_new": torch.zeros(2, 2, 256, dtype=_BF)}, TypeError, "share q_gate's dtype"),
    ({"v_pages": torch.zeros(3, 16, 2, 256, dtype=_BF)}, ValueError, "k_pages and v_pages must be"),     # fewer pages than K's
    ({"v_pages": torch.zeros(5, 16, 2, 256, dtype=_BF)}, ValueError, "k_pages and v_pages must be"),
    ({"v_pages": torch.zeros(4, 8, 2, 256, dtype=_BF)}, ValueError, "k_pages and v_pages must be"),
    ({"k_pages": torch.zeros(4, 16, 256, 2, dtype=_BF), "v_pages": torch.zeros(4, 16, 256, 2, dtype=_BF)}, ValueError, "k_pages and v_pages must be"),
    ({"k_pages": torch.zeros(64, 2, 256, dtype=_BF), "v_pages": torch.zeros(64, 2, 256, dtype=_BF)}, ValueError, "k_pages and v_pages must be"),
    ({"q_gate": torch.zeros(2, 16, 511)}, ValueError, "q_gate must be"),
    ({"k_new": torch.zeros(3, 2, 256)}, ValueError, "q_gate must be"),
    ({"v_new": torch.zeros(2, 2, 255)}, ValueError, "q_gate must be"),
    ({"params": {"q_norm_w": torch.ones(255), "k_norm_w": torch.ones(256)}}, ValueError, _NORMS),
    ({"params": {"q_norm_w": torch.ones(256), "k_norm_w": torch.ones(128)}}, ValueError, _NORMS),
    ({"params": {"q_norm_w": torch.ones(256, dtype=_BF), "k_norm_w": torch.ones(256)}}, TypeError, "q_norm_w must be torch.float32"),
    ({"table": torch.zeros(2, 2, dtype=torch.int64)}, TypeError, "the page table must be torch.int32"),
    ({"out": torch.zeros(1, 16, 256)}, ValueError, "out must be"),
    ({"out": torch.zeros(2, 16, 512)[:, :, ::2]}, ValueError, "out must be contiguous"),
    ({"out": torch.zeros(2, 16, 256, dtype=torch.float64)}, TypeError, "unsupported dtype"),
    ({"q_gate": torch.zeros(2, 16, 1024)[:, :, ::2]}, ValueError, "q_gate must be contiguous"),
    ({"k_new": torch.zeros(2, 2, 512)[:, :, ::2]}, ValueError, "k must be contiguous"),
    ({"v_new": torch.zeros(2, 2, 512)[:, :, ::2]}, ValueError, "v must be contiguous"),
    ({"k_pages": torch.zeros(8, 16, 2, 256, dtype=_BF)[::2]}, ValueError, "k_pages must be contiguous"),
    ({"v_pages": torch.zeros(8, 16, 2, 256, dtype=_BF)[::2]}, ValueError, "v_pages must be contiguous")])
def test_each_wrapper_check_by_itself(on_host, change, error, match):
    """What the wrapper lets through without this one check, it refuses with
    the check's own message, in all three calls; nothing reaches the library."""
    from qff import ops
    ctx, calls = on_host
    for name, call in _each_call(ops, ctx, {**_args(), **change}):
        with pytest.raises(error, match=match):
            call()
    assert not calls.made


def test_table_and_sequence_checks_by_themselves(on_host):
    from qff import ops
    ctx, calls = on_host
    a = _args()
    ints = lambda *n: torch.zeros(*n, dtype=torch.int32)   # noqa: E731
    for table in (ints(3, 2), ints(1, 2), ints(2), ints(2, 2, 1)):
        with pytest.raises(ValueError, match=r"the page table must be \[2, entries\]"):
            ops.gqa_decode_paged(ctx, **{**a, "table": table})
    with pytest.raises(ValueError, match="the page table must be contiguous"):
        ops.gqa_decode_paged(ctx, **{**a, "table": ints(2, 4)[:, ::2]})
    for positions in (ints(1), ints(3)):
        with pytest.raises(ValueError, match="positions must be"):
            ops.gqa_decode_paged(ctx, **{**a, "positions": positions})
    with pytest.raises(TypeError, match="positions must be torch.int32"):
        ops.gqa_decode_paged(ctx, **{**a, "positions": torch.zeros(2, dtype=torch.int64)})
    for more in ({"group": ints(1), "shared_len": ints(2)}, {"group": ints(2), "shared_len": ints(3)}):
        with pytest.raises(ValueError, match="positions, group and shared_len must be"):
            ops.gqa_decode_shared(ctx, **a, **more)
    for name in ("group", "shared_len"):
        with pytest.raises(TypeError, match=f"{name} must be torch.int32"):
            ops.gqa_decode_shared(ctx, **a, **{"group": ints(2), "shared_len": ints(2), name: torch.zeros(2)})
    one = {"params": a["params"], "q_gate": a["q_gate"], "k": a["k_new"], "v": a["v_new"], "k_pages": a["k_pages"], "v_pages": a["v_pages"]}
    for table in (ints(2, 2), ints(1, 1, 2)):
        with pytest.raises(ValueError, match=r"the page table must be \[1, entries\]"):
            ops.gqa_prefill_paged(ctx, **one, table=table)
    with pytest.raises(TypeError, match="the page table must be torch.int32"):
        ops.gqa_prefill_paged(ctx, **one, table=torch.zeros(2, dtype=torch.int64))
    assert not calls.made
    # another device than the context's
    far = types.SimpleNamespace(device=0, handle=None)
    for name, call in _each_call(ops, far, a):
        with pytest.raises(ValueError, match="must live on the context's device, cuda:0"):
            call()
    assert not calls.made


def test_copy_wrapper_checks_by_themselves(on_host):
    from qff import ops
    ctx, calls = on_host
    pool = torch.zeros(4, 16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)   # noqa: E731
    for pools, src, dst, error, match in (
            ([], [0], [1], ValueError, "at least one pool"),
            ([pool], [0, 1], [2], ValueError, "src and dst must have the same length"),
            ([pool], [0], [], ValueError, "src and dst must have the same length"),
            ([pool, pool[:3]], [0], [1], ValueError, "the same number of pages"),
            ([pool, torch.zeros(4, 12)], [0], [1], ValueError, "the same number of pages"),
            ([pool, torch.zeros(8, 8)], [0], [1], ValueError, "the same number of pages"),     # as many bytes, other pages
            ([pool, torch.zeros(4, 32)[:, ::2]], [0], [1], ValueError, "a pool must be contiguous"),
            ([pool], torch.tensor([0]), i32(1), TypeError, "src must be"),
            ([pool], i32(0), torch.tensor([1]), TypeError, "dst must be"),
            ([pool], i32(0)[None], i32(1), TypeError, "src must be"),
            ([pool], i32(0, 0, 1, 1)[::2], i32(2, 3), TypeError, "src must be")):
        with pytest.raises(error, match=match):
            ops.pages_copy(ctx, pools, src, dst)
    with pytest.raises(ValueError, match="must live on the context's device, cuda:0"):
        ops.pages_copy(types.SimpleNamespace(device=0, handle=None), [pool], [0], [1])
    assert not calls.made


def _program(tmp_path, name):
    """A C++ program of tests/host_checks over the library, built with g++."""
    from qff._lib import LIB_PATH
    exe, rocm = str(tmp_path / name), os.environ.get("ROCM_PATH", "/opt/rocm")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-w", "-I" + os.path.join(rocm, "include"),
                        "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "qwen-fieldfare_amd", "csrc"),
                        os.path.join(ROOT, "tests", "host_checks", name + ".cpp"), LIB_PATH, "-L" + os.path.join(rocm, "lib"),
                        "-lamdhip64", "-Wl,-rpath," + os.path.dirname(LIB_PATH), "-Wl,-rpath," + os.path.join(rocm, "lib"),
                        "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return exe


def test_split_of_short_slices(tmp_path):
    """The shapes that tests/test_gpu_paged_blocks.py means for blocks of 16 tokens
    take them; for slices of any length behind any history, in contexts of few
    partial rows too, the split keeps to its workgroups and partial rows."""
    import random

    import test_gpu_paged_blocks as blocks
    import qff
    qff.lib()
    exe = _program(tmp_path, "paged_split")
    C, P = blocks.CONTEXT["max_ctx"], blocks.CONTEXT["max_prefill_tokens"]
    tokens = blocks.BLOCKS_OF_16 + blocks.BLOCKS_OF_8
    assert sum(t <= 42 for _, t in blocks.BLOCKS_OF_16) >= 5    # (as many tokens as three terms take)
    rng = random.Random(1)
    more = []
    for _ in range(3000):
        t = rng.randint(1, 64)
        c = int(2 ** rng.uniform(7, 17))
        more.append((c, rng.choice([t, 64, 8192]), rng.randint(0, max(0, c - t)), t))
    r = subprocess.run([exe], input="\n".join(" ".join(map(str, x)) for x in [(C, P, s, t) for s, t in tokens] + more),
                       capture_output=True, text=True)
    assert r.returncode == 0, [line for line in r.stdout.splitlines() if "BAD" in line][:5]
    lines = r.stdout.splitlines()
    assert len(lines) == len(tokens) + len(more)
    for shape, line in zip(tokens, lines):
        assert line.split()[0] == ("16" if shape in blocks.BLOCKS_OF_16 else "8"), (shape, line)


def test_a_contexts_limits_hold_what_zeros_stand_for(monkeypatch):
    """What checks against ctx.cfg see is what the library applies."""
    from qff import ops
    made = []
    monkeypatch.setattr(ops, "lib", lambda: types.SimpleNamespace(qff_ctx_create=lambda h, device, cfg: made.append(cfg) or 0))
    for args, want in (((0, 0, 0, 0), (32, 65536, 8192)), ((0, 4, 0, 16), (4, 65536, 16)), ((0,), (32, 65536, 8192))):
        c = ops.Context(*args)
        assert (c.cfg.max_batch, c.cfg.max_ctx, c.cfg.max_prefill_tokens) == want
        c.handle = None
    assert len(made) == 3


def test_copy_launches_stay_within_a_grid(tmp_path):
    import qff
    qff.lib()
    r = subprocess.run([_program(tmp_path, "copy_launches")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-1000:]
