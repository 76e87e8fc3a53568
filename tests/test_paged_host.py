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
