"""Bounded waits of the tensor-core attention kernels, without a GPU fault: the test hook
leaves one copy of every block unissued, so the waits on it run out.  The kernel returns,
the host sees NSC_ERR_TIMEOUT, and a clean run afterwards is correct."""

import pytest
import torch

import neural_shift_cuda_b200 as nsc
from neural_shift_cuda_b200 import _lib
from oracle import token_oracle as T
from token_cases import check, leaf, randn, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("skip", [0, 2])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("part", ["forward", "backward"])
def test_skipped_copy_times_out_and_context_survives(cuda, part, D, skip):
    L = 400
    q, k, v, go = (leaf(randn(i, 1, L, 2, D, dtype=torch.bfloat16).to(cuda)) for i in range(4))

    def step(fault=None):
        """A training step; the fault is in force for its one half."""
        try:
            if fault == "forward":
                _lib.test_wait_fault(skip, 4)
            out = nsc.token_attention(q, k, v, causal=True)
            if fault == "backward":
                _lib.test_wait_fault(skip, 4)
            grads = torch.autograd.grad(out, [q, k, v], go.detach())
            if fault:
                with pytest.raises(RuntimeError, match="NSC_ERR_TIMEOUT"):
                    _lib.check_device_waits()
        finally:
            _lib.test_wait_fault(-1, 0)
        return out, grads

    step()
    _lib.check_device_waits()
    before = _lib.wait_timeouts()
    step(part)
    assert _lib.wait_timeouts() > before
    out, grads = step()
    _lib.check_device_waits()
    want = reference(q, k, v, T.visible(1, L, L, True), go, D ** -0.5)
    check(out, want[0], torch.bfloat16, "out")
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"), grads, want[2:5]):
        check(g, w, torch.bfloat16, name)
