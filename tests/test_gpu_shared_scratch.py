"""The chunked DeltaNet prefill, the expert block and sampling have their scratch in the same bytes of the context's
workspace: each call's results are those of a context of its own, whatever the others left there."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV, bf16_tensor, f32_tensor
from qff import synth
from test_gpu_moe import _handle, _indices, _weights

pytestmark = pytest.mark.gpu


def test_calls_in_turn(hip):
    import qff
    rng = np.random.default_rng(0)
    cfg = dict(max_batch=8, max_ctx=256, max_prefill_tokens=256)
    E, top, D, I, n = 6, 4, 512, 128, 200
    w = _handle(_weights(rng, E, D, I, "bf16", True))
    x = torch.from_numpy(rng.standard_normal((n, D))).float().to(DEV)
    idx = torch.from_numpy(_indices(rng, n, E, top, "any")).to(DEV)
    sc = torch.rand(n, top, device=DEV)
    logits, u = torch.randn(8, 30000, device=DEV), torch.rand(8, device=DEV)
    settings = dict(top_k=torch.tensor([0, 1, 40, 29999, 7, 0, 100, 0], dtype=torch.int32, device=DEV),
                    top_p=torch.tensor([1, .9, .5, .999, .1, .7, 1, .3], device=DEV))
    T = 150
    prm = {k: f32_tensor(v) for k, v in synth.deltanet_params().items()}
    bf = lambda *s: bf16_tensor((rng.standard_normal(s).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16))   # noqa: E731
    qkv, z = bf(T, 8192), bf(T, 4096)
    a, b = (torch.randn(T, 32, device=DEV) for _ in range(2))

    def nan(ctx):   # pairs' rows, factors and sums that are no numbers, all over the shared bytes
        h = torch.full((256, top + 1, 2048), float("nan"), device=DEV)
        big = _handle(_weights(np.random.default_rng(1), 2, 2048, 64, "bf16", True), "down", "shared_down")
        out = qff.moe_down(ctx, big, h[:, :, :64].contiguous(), torch.zeros(256, top, dtype=torch.int32, device=DEV),
                           torch.ones(256, top, device=DEV))
        assert out.isnan().all()
        return []

    def moe(ctx):
        h = qff.moe_gate_up(ctx, w, x, idx)
        return [h, qff.moe_down(ctx, w, h, idx, sc, residual=x), qff.moe_down(ctx, w, h.half(), idx, sc, out_dtype=torch.bfloat16)]

    def sample(ctx):
        return list(qff.sample(ctx, logits, u, **settings))

    def prefill(ctx):
        conv, ssm = torch.zeros(8192, 4, device=DEV), torch.zeros(32, 128, 128, device=DEV)
        return [qff.deltanet_prefill(ctx, prm, qkv, z, a, b, conv, ssm), conv, ssm]

    calls = [moe, sample, prefill, nan]
    alone = {}
    for f in calls:
        ctx = qff.Context(**cfg)
        alone[f] = f(ctx)
        torch.cuda.synchronize()
        ctx.close()
    ctx = qff.Context(**cfg)
    for order in ([3, 2, 0, 1, 2], [3, 0, 2, 1, 0], [3, 1, 0, 3, 1, 2]):
        for i in order:
            print("call", calls[i].__name__, flush=True)
            got = calls[i](ctx)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, alone[calls[i]], strict=True)), calls[i].__name__
    ctx.close()
