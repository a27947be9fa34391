"""What the token-attention operators refuse, and the bucket map; no GPU."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad as fwd

import neural_shift_cuda_b200 as nsc
from neural_shift_cuda_b200 import _lib


def _qkv(B=1, L=4, Hq=2, Hkv=1, D=8, dt=torch.float32):
    return (torch.zeros(B, L, Hq, D, dtype=dt), torch.zeros(B, L, Hkv, D, dtype=dt),
            torch.zeros(B, L, Hkv, D, dtype=dt))


def test_cpu_tensors_are_refused():
    q, k, v = _qkv()
    cos = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nsc.token_attention(q, k, v)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nsc.token_attention_decode(q, k, v, torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        nsc.qk_norm_rotate(q, k, None, None, cos, cos)


@pytest.mark.parametrize("change,err,match", [
    (dict(q=torch.zeros(4, 2, 8)), RuntimeError, "must be"),
    (dict(k=torch.zeros(1, 4, 1, 16)), RuntimeError, "do not agree"),
    (dict(v=torch.zeros(1, 5, 1, 8)), RuntimeError, "do not agree"),
    (dict(k=torch.zeros(1, 4, 3, 8), v=torch.zeros(1, 4, 3, 8)), RuntimeError, "multiple"),
    (dict(k=torch.zeros(1, 4, 1, 8).half()), TypeError, "float16"),
    (dict(q=torch.zeros(1, 4, 2, 8).long(), k=torch.zeros(1, 4, 1, 8).long(),
          v=torch.zeros(1, 4, 1, 8).long()), TypeError, "unsupported"),
    (dict(prefix=3), ValueError, "causal"),
    (dict(bias_table=torch.zeros(4, 2)), ValueError, "bias_buckets"),
    (dict(bias_buckets=torch.zeros(3, dtype=torch.int32)), ValueError, "bias_table"),
    (dict(bias_table=torch.zeros(4, 3), bias_buckets=torch.zeros(3, dtype=torch.int32)),
     RuntimeError, "bias_table"),
    (dict(bias_table=torch.zeros(4, 2), bias_buckets=torch.zeros(4, dtype=torch.int32)),
     RuntimeError, "2 reach"),
    (dict(bias_table=torch.zeros(4, 2), bias_buckets=torch.zeros(3)), TypeError, "int32"),
    (dict(bias_table=torch.zeros(4, 2).double(),
          bias_buckets=torch.zeros(3, dtype=torch.int32)), TypeError, "bias_table"),
])
def test_attention_refusals(change, err, match):
    q, k, v = _qkv()
    args = dict(q=q, k=k, v=v)
    args.update(change)
    with pytest.raises(err, match=match):
        nsc.token_attention(**args)


def test_decode_refuses_gradients():
    q, k, v = _qkv()
    with pytest.raises(RuntimeError, match="no backward"):
        nsc.token_attention_decode(q.requires_grad_(), k, v, torch.ones(1, dtype=torch.int32))


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_tangents_are_refused(no_grad):
    """Dropped, they would give a derivative of zero without a word."""
    q, k, v = _qkv()
    table, m = torch.zeros(4, 2), torch.zeros(3, dtype=torch.int32)
    n, cos, w = torch.ones(1, dtype=torch.int32), torch.zeros(4, 4), torch.zeros(8)
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        bias = dict(bias_table=dual(table), bias_buckets=m)
        for call in (lambda: nsc.token_attention(dual(q), k, v),
                     lambda: nsc.token_attention(q, k, dual(v)),
                     lambda: nsc.token_attention(q, k, v, **bias),
                     lambda: nsc.token_attention_decode(q, dual(k), v, n),
                     lambda: nsc.token_attention_decode(q, k, v, n, **bias),
                     lambda: nsc.qk_norm_rotate(q, dual(k), None, None, cos, cos),
                     lambda: nsc.qk_norm_rotate(q, k, dual(w), None, cos, cos),
                     lambda: nsc.qk_norm_rotate(q, k, None, None, cos, dual(cos))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # (tensors without tangents pass this check inside a level too)
        with pytest.raises(RuntimeError, match="no CPU path"):
            nsc.token_attention(q, k, v)


def test_rotate_refusals():
    q, k, _ = _qkv()
    cos = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="do not agree"):
        nsc.qk_norm_rotate(q, k[:, :3], None, None, cos, cos)
    with pytest.raises(RuntimeError, match="q_weight"):
        nsc.qk_norm_rotate(q, k, torch.zeros(7), None, cos, cos)
    with pytest.raises(TypeError, match="q_weight"):
        nsc.qk_norm_rotate(q, k, torch.zeros(8).half(), None, cos, cos)
    with pytest.raises(RuntimeError, match="cos and sin"):
        nsc.qk_norm_rotate(q, k, None, None, torch.zeros(4, 5), torch.zeros(4, 5))


def _att(**kw):
    a = _lib.Attention()
    base = dict(B=1, Lq=4, Lk=4, Hq=2, Hkv=1, D=8, scale=1.0, dtype=2)
    base.update(kw)
    for n, x in base.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change,status,match", [
    (dict(), 1, "NULL"),
    (dict(dtype=9), 2, "dtype"),
    (dict(D=257), 1, "exceeds"),
    (dict(D=129, dtype=3), 1, "exceeds"),
    (dict(Hq=3, Hkv=2), 1, "multiple"),
    (dict(Lk=1 << 31), 1, "too many"),
    (dict(softcap=-1.0), 1, "softcap"),
    (dict(softcap=float("nan")), 1, "softcap"),
    (dict(table=16), 1, "table and its buckets"),
    (dict(table=16, buckets=16, n_buckets=257, table_dtype=2), 1, "buckets"),
    (dict(table=16, buckets=16, n_buckets=8, reach=1025, table_dtype=2), 1, "reach"),
    (dict(table=16, buckets=16, n_buckets=8, reach=5, table_dtype=1), 2, "bias table"),
    (dict(prefix=16), 1, "causal"),
    (dict(documents=16, docs=1, Lq=3), 1, "documents"),
])
def test_entry_point_refusals(change, status, match):
    """Before any device is touched: the addresses here are not real."""
    lib = _lib.load()
    a = _att(**change)
    assert lib.nsc_token_attention_fwd(ctypes.byref(a), *[None] * 5) == status
    assert match in lib.nsc_last_error_string().decode()
    g = _lib.AttentionGrad()
    assert lib.nsc_token_attention_bwd(ctypes.byref(a), ctypes.byref(g), None) == status
    assert lib.nsc_token_attention_fwd(*[None] * 6) == 1


def test_empty_calls_are_noops():
    lib = _lib.load()
    a = _att(B=0)
    assert lib.nsc_token_attention_fwd(ctypes.byref(a), *[None] * 5) == 0
    a = _att(B=0, causal=1)
    assert lib.nsc_token_attention_decode(ctypes.byref(a), None, None, None, None) == 0
    n = _lib.NormRotate()
    n.D, n.dtype = 8, 2
    assert lib.nsc_qk_norm_rotate_fwd(ctypes.byref(n), None, None, None) == 0
    n.D = 7
    assert lib.nsc_qk_norm_rotate_fwd(ctypes.byref(n), None, None, None) == 1
    assert lib.nsc_qk_norm_rotate_workspace(ctypes.byref(n)) == -1


@pytest.mark.parametrize("cap", [1e-31, 1e-300, 1e31, float("inf")])
def test_caps_that_32_bits_do_not_hold_are_refused(cap):
    lib = _lib.load()
    a = _att(softcap=cap, causal=1)
    for st in (lib.nsc_token_attention_fwd(ctypes.byref(a), *[None] * 5),
               lib.nsc_token_attention_decode(ctypes.byref(a), *[None] * 4)):
        assert st == 1 and "softcap" in lib.nsc_last_error_string().decode()
    assert lib.nsc_token_attention_bwd_workspace(ctypes.byref(a)) == -1


def test_decode_of_more_rows_than_a_grid_has_is_refused():
    lib = _lib.load()
    a = _att(B=4096, Hq=16, Hkv=16, Lq=1 << 15, Lk=4096, D=8, dtype=0, causal=1,
             q=256, k=256, v=256)
    assert lib.nsc_token_attention_decode(ctypes.byref(a), 256, None, 256, None) == 1
    assert "too many" in lib.nsc_last_error_string().decode()


def test_workspaces_that_are_not_aligned_are_refused():
    lib = _lib.load()
    a = _att(causal=1, q=256, k=256, v=256)
    assert lib.nsc_token_attention_decode(ctypes.byref(a), 256, None, 264, None) == 1
    assert "aligned" in lib.nsc_last_error_string().decode()
    g = _lib.AttentionGrad()
    for n in ("out", "stats", "grad_out", "grad_q", "grad_k", "grad_v"):
        setattr(g, n, 256)
    g.workspace = 264
    assert lib.nsc_token_attention_bwd(ctypes.byref(a), ctypes.byref(g), None) == 1
    assert "aligned" in lib.nsc_last_error_string().decode()


def test_relative_buckets():
    m = nsc.relative_buckets(8, 6)
    assert m.dtype == torch.int32 and m.tolist() == [3, 3, 3, 2, 2, 1, 0, 5, 6, 6, 7, 7, 7]
    m = nsc.relative_buckets(4, 8, bidirectional=False)
    assert m.tolist() == [3, 3, 3, 3, 3, 2, 2, 1, 0] + [0] * 8
    m = nsc.relative_buckets(32, 128)
    assert m.shape == (257,) and int(m.max()) == 31 and int(m[128]) == 0
    assert (m[:128].diff() <= 0).all() and (m[129:].diff() >= 0).all()
    for bad in ((2, 5), (300, 500), (32, 8), (32, 2000)):
        with pytest.raises(ValueError):
            nsc.relative_buckets(*bad)
