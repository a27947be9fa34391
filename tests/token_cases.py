"""Shared by the token-attention tests: inputs, the 64-bit results, and bounds.

A result in a type of unit roundoff u is held to 3 u of its norm: one rounding
of the output, one of the softmax weights or score gradients before the second
product, one unit of slack.  In fp32 the error is that of the scores: a dot
product of D terms and an exponent up to about 30 give some 30 u each way, so
64 u (fp64: the same).  Single elements may be 24 u (fp32, fp64: 512 u) of the
largest value off.
"""

import torch

from oracle import token_oracle as T

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24,
     torch.float64: 2.0 ** -53}


def check(got, want, dt, what="", grow=1.0):
    want = want.detach().double().cpu()
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(got)), what
    assert torch.equal(want[~fin].nan_to_num(7.0), got[~fin].nan_to_num(7.0)), what
    d, w = (got - want)[fin], want[fin]
    if not w.numel():
        return
    exact = dt in (torch.float32, torch.float64)
    u = U[dt] * grow
    norm = (64 if exact else 3) * u
    most = (512 if exact else 24) * u
    size = float(w.norm())
    assert float(d.norm()) <= norm * size + 1e-300, \
        f"{what}: {float(d.norm()) / max(size, 1e-300):.3g} of the norm, {norm:.3g} allowed"
    assert float(d.abs().max()) <= most * float(w.abs().max()) + 1e-300, \
        f"{what}: element off by {float(d.abs().max()):.3g} of {float(w.abs().max()):.3g}"


def randn(seed, *shape, dtype, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * mul).to(dtype)


def leaf(t):
    return None if t is None else t.detach().requires_grad_()


def reference(q, k, v, seen, gout, scale, cap=0.0, table=None, buckets=None, glse=None):
    """(out, lse, dq, dk, dv, dtable) in fp64 on the tensors' device."""
    q, k, v, table = (leaf(None if t is None else t.double()) for t in (q, k, v, table))
    out, lse = T.attention(q, k, v, seen, scale, cap, table, buckets)
    loss = (out * gout.double()).sum()
    if glse is not None:
        loss = loss + (torch.where(torch.isfinite(lse), lse, 0.0) * glse.double()).sum()
    ins = [q, k, v] + ([table] if table is not None else [])
    g = torch.autograd.grad(loss, ins, allow_unused=True)
    g = [torch.zeros_like(i) if x is None else x for x, i in zip(g, ins)]
    return out.detach(), lse.detach(), g[0], g[1], g[2], (g[3] if table is not None else None)
