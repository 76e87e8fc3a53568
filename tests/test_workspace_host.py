"""What a context's workspace holds, from its size alone, and what a large one does not allow."""
import ctypes
import subprocess

from test_paged_host import _program


def _size(*cfg):
    import qff
    from qff._lib import CtxCfg
    n = ctypes.c_size_t()
    assert qff.lib().qff_workspace_size(ctypes.byref(CtxCfg(*cfg)), ctypes.byref(n)) == 0
    return n.value


def test_scratch_of_one_call_is_shared():
    """Expert block and sampling lie in the bytes of the chunked prefill's records. At the defaults those are the most:
    per 64 tokens and 16 key heads K and Q, per 32 value heads T, P, gates and beta V; what stands beside them is the attention's
    and the Q4 products' own, and prefill rows of [T][4096] fp32."""
    records = 8192 // 64 * (16 * (2 * 64 * 128 + 2 * 16 * 512) * 2 + 32 * (2 * 6 * 512 * 2 * 2 + 4 * 64 * 4 + 64 * 128 * 4))
    slots, partials = max(32, 4) * 2 * 128, 8192 * (4096 + 32) * 4
    attention = slots * 8 * (2 + 256) * 4 + 8192 * 4096 * 2 + 2 * 65536 * 1024
    products = 8192 * 4096 * 2 + 8192 * 4 + 4096 * 16 * 64 * 4
    assert 0 <= _size(32, 65536, 8192) - (records + partials + attention + products) < 1 << 16   # (counters, rounding to 256 bytes)


def test_many_sequences_cost_what_sampling_lists():
    """One more sequence: a list of 262144 int32, 65 chunks' bins of 256 weights, and less than 64 KB beside (its share
    of the attention's partials 2 MB)."""
    per = (_size(2064, 64, 1) - _size(2063, 64, 1)) - 2 * 128 * 8 * (2 + 256) * 4
    assert 0 <= per - (262144 * 4 + 65 * 256 * 8) < 1 << 16


def test_batches_that_sampling_refuses(tmp_path):
    """A context whose max_batch is more than a grid's second dimension holds."""
    import qff
    qff.lib()
    r = subprocess.run([_program(tmp_path, "sample_batch")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
