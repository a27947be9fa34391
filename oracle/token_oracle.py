"""Plain 64-bit forms of the token-attention operators, on the CPU or a GPU.

Written from the definitions with dense masks and torch autograd; test
infrastructure only.  A query that sees nothing gives zeros, and values that a
query does not see are replaced by zeros before any product, so that they
cannot reach it even where they are not finite.
"""

from __future__ import annotations

import math

import torch


def qk_norm_rotate(q, k, wq, wk, cos, sin, positions=None, adjacent=False, eps=1e-6):
    def one(x, w):
        x = x.double()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.double()
        at = (torch.arange(x.shape[1], device=x.device).expand(x.shape[:2])
              if positions is None else positions.long().expand(x.shape[:2]))
        c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
        R = 2 * cos.shape[1]
        t, rest = y[..., :R], y[..., R:]
        if adjacent:
            a, b = t[..., 0::2], t[..., 1::2]
            t = torch.stack([a * c - b * s, a * s + b * c], -1).reshape(t.shape)
        else:
            a, b = t[..., :R // 2], t[..., R // 2:]
            t = torch.cat([a * c - b * s, a * s + b * c], -1)
        return torch.cat([t, rest], -1)
    return one(q, wq), one(k, wk)


def visible(B, Lq, Lk, causal=False, prefix=None, documents=None, lengths=None):
    """(B, Lq, Lk) bool: which keys each query sees, pair by pair."""
    seen = torch.zeros(B, Lq, Lk, dtype=torch.bool)
    for b in range(B):
        n = Lk if lengths is None else int(lengths[b])
        groups = ([(0, n)] if documents is None else
                  [(int(documents[b][d]), int(documents[b][d + 1]))
                   for d in range(len(documents[b]) - 1)])
        pos = torch.arange(Lq)[:, None] + (n - Lq)
        key = torch.arange(Lk)[None, :]
        for d, (s, e) in enumerate(groups):
            ok = (key >= s) & (key < e)
            if documents is not None:
                ok = ok & (pos >= s) & (pos < e)
            if causal:
                pre = 0 if prefix is None else int(prefix[b][d])
                ok = ok & ((key <= pos) | (key < s + pre))
            seen[b] |= ok
    return seen


def _finite(t):
    return torch.where(torch.isinf(t), torch.zeros_like(t), t)


def attention(q, k, v, seen, scale, softcap=0.0, table=None, buckets=None, offset=None):
    """(out, lse) in fp64; `seen` (B, Lq, Lk); offset (B,): the position of
    query 0 (default Lk - Lq)."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    dev = q.device
    seen = seen.to(dev)
    kk = k.double().repeat_interleave(Hq // Hkv, 2)
    vv = v.double().repeat_interleave(Hq // Hkv, 2)
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), kk) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if table is not None:
        reach = buckets.shape[0] // 2
        if offset is None:
            offset = torch.full((B,), Lk - Lq)
        rel = (torch.arange(Lk)[None, None, :] - torch.arange(Lq)[None, :, None]
               - offset.cpu()[:, None, None]).to(dev)
        at = buckets.long()[rel.clamp(-reach, reach) + reach]
        # as a product, so that the table's gradient is a blocked sum and not
        # a chain of single additions, whose rounding shows in 64 bits
        pick = (at[..., None] == torch.arange(table.shape[0], device=dev)).double()
        s = s + (pick @ _finite(table.double())).permute(0, 3, 1, 2)
        for u in torch.nonzero((table == -math.inf).any(1)).flatten().tolist():
            gone = (table[u] == -math.inf)[None, :, None, None] & (at == u)[:, None]
            s = s.masked_fill(gone, -math.inf)
    hide = ~seen[:, None]
    s = s.masked_fill(hide, -math.inf)
    top = s.detach().amax(-1, keepdim=True) if Lk else s.new_zeros(B, Hq, Lq, 1)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top).masked_fill(hide, 0.0)
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total[..., 0] == 0, torch.full_like(total[..., 0], -math.inf),
                      top[..., 0] + torch.log(torch.where(
                          total[..., 0] == 0, torch.ones_like(total[..., 0]), total[..., 0])))
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.einsum("bhqk,bkhd->bqhd", p, vv)
    return out, lse
