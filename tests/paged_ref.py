"""Plain restatement, in 64 bits, of the paged full-attention calls: one
sequence at a time, the cache rows gathered through the table. The attention
reads the rows as the cache holds them."""
import math

import torch


def rope_norm(x, w, pos, theta=1e7, eps=1e-6):
    """Head RMS norm and rotation of the first 64 dims of x [n, heads, 256] at
    positions [n]; angles are fp32 products of fp32 inverse frequencies."""
    x = x.double()
    x = x / torch.sqrt(x.square().mean(2, keepdim=True) + eps) * w.double()
    e = torch.arange(32, dtype=torch.float32) * 2 / 64
    f = (1.0 / torch.pow(torch.tensor(theta, dtype=torch.float32), e)).to(x.device)
    ang = (pos.float()[:, None] * f[None, :]).double()[:, None, :]
    lo, hi = x[:, :, :32], x[:, :, 32:64]
    return torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin(), x[:, :, 64:]], 2)


def rows_of(pages, table_row, n):
    """The first n positions' rows [n, 2, 256] of a sequence, in 64 bits."""
    page = pages.shape[1]
    at = torch.arange(n, device=pages.device)
    return pages[table_row.long()[at // page], at % page].double()


def attend(params, q_gate, k_pages, v_pages, table_row, pos, scale=1.0 / 16, **rope):
    """Tokens q_gate [n, 16, 512] of one sequence at positions pos [n], each
    over positions 0 .. pos of the cache as it stands -> [n, 16, 256]."""
    n, last = q_gate.shape[0], int(pos.max())
    q = rope_norm(q_gate[:, :, :256], params["q_norm_w"], pos, **rope)
    K, V = rows_of(k_pages, table_row, last + 1), rows_of(v_pages, table_row, last + 1)
    hidden = torch.arange(last + 1, device=pos.device)[None, :] > pos[:, None]
    out = torch.empty(n, 16, 256, dtype=torch.float64, device=q_gate.device)
    for h in range(16):
        s = (q[:, h].contiguous() @ K[:, h // 8].t().contiguous()) * scale
        out[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ V[:, h // 8].contiguous()
    return out * torch.sigmoid(q_gate[:, :, 256:].double())
