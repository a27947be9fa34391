"""Edges of the token operators: what lands late, what nothing sees, what is not aligned,
and values near the ends of their type."""

import math

import pytest
import torch

import neural_shift_cuda_b200 as nsc
from oracle import token_oracle as T
from token_cases import check, leaf, randn, reference

pytestmark = pytest.mark.gpu

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 64), (BF16, 128), (F16, 128)])
def test_gradients_while_memory_is_busy(cuda, dt, D):
    """Every product waits for its own operands: the gradients have the same bits when
    copies on another stream hold the output gradient's tiles back."""
    q, k, v, go = (randn(i, 2, 640, 8, D, dtype=dt).to(cuda) for i in range(4))
    want = reference(q, k, v, T.visible(2, 640, 640), go, D ** -0.5)[2:5]
    leaves = [leaf(t) for t in (q, k, v)]
    out = nsc.token_attention(*leaves)
    quiet = torch.autograd.grad(out, leaves, go, retain_graph=True)
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"), quiet, want):
        check(g, w, dt, name)
    # (each copy is larger than the L2 cache, so that tiles come from memory too)
    src, dst = (torch.empty(1 << 28, dtype=torch.uint8, device=cuda) for _ in range(2))
    side = torch.cuda.Stream()
    for _ in range(8):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                dst.copy_(src)
        busy = torch.autograd.grad(out, leaves, go, retain_graph=True)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(quiet, busy):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D", [16, 32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_short_rows_and_values_that_are_not_finite(cuda, dt, D, bad):
    """Two blocks of keys: a bad value of the first shows in every query that sees it, in
    every head, and in no other; so does one of the second."""
    L, at = 128, (3, 100)
    q, k, v = (randn(i, 16, L, 8, D, dtype=dt).to(cuda) for i in range(3))
    want = nsc.token_attention(q, k, v, causal=True)
    for key in at:
        v2 = v.clone()
        v2[:, key] = bad
        for _ in range(10):
            got = nsc.token_attention(q, k, v2, causal=True)
            assert torch.equal(got[:, :key], want[:, :key])
            assert not torch.isfinite(got[:, key:]).any()
