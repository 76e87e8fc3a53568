"""qff_sample's results do not depend on how a row is cut up: rows of a large batch (8 chunks each, of up to 32768 tokens)
against the same rows alone (64 chunks) and in a middle-sized batch, bit for bit; a few of them against the definition."""
import numpy as np
import pytest
import torch

import moe_ref as R
from gpu_util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,dtype", [(262144, torch.bfloat16), (151936, torch.float32), (513, torch.float32)])
def test_rows_alone_and_in_batches(hip, vocab, dtype):
    import qff
    print("sample", vocab, dtype, flush=True)
    B = 130
    ctx = qff.Context(max_batch=B, max_ctx=64, max_prefill_tokens=1)
    rng = np.random.default_rng(vocab)
    l = (torch.randn(B, vocab, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) * 3).to(dtype)
    l[3] = 0.0                      # ties all over, borders among them
    l[4] = -float("inf")
    l[5, ::2] = -float("inf")
    host = {"u": rng.random(B), "temperature": rng.uniform(0.2, 2, B) * (rng.random(B) < 0.9), "top_k": rng.integers(0, 3, B) * rng.integers(1, vocab, B),
            "top_p": np.where(rng.random(B) < 0.5, 1.0, rng.uniform(0.1, 1, B)), "min_p": np.where(rng.random(B) < 0.7, 0.0, rng.uniform(0.001, 0.3, B))}
    dev = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device=DEV) for k, v in host.items()}

    def run(rows):
        tok, prob = qff.sample(ctx, l[rows].contiguous(), **{k: v[rows].contiguous() for k, v in dev.items()})
        torch.cuda.synchronize()
        return tok, prob

    tok, prob = run(slice(0, B))
    for rows in [slice(i, i + 1) for i in range(0, B, 7)] + [slice(3, 4), slice(4, 5), slice(5, 6), slice(0, 40), slice(90, B)]:
        a, b = run(rows)
        assert torch.equal(a, tok[rows]) and torch.equal(b, prob[rows]), rows
    for i in (0, 3, 4, 5, 129):
        v = {k: float(x[i]) for k, x in host.items()}
        ref = R.sample_row(l[i].float().cpu().numpy(), v["u"], v["temperature"], int(v["top_k"]), v["top_p"], v["min_p"])
        assert int(tok[i]) == ref[0] and abs(float(prob[i]) - ref[1]) <= 2 ** -23 * ref[1], (i, int(tok[i]), float(prob[i]), ref)
    ctx.close()
