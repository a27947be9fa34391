"""Edges of the token operators: what lands late, what nothing sees, what is not aligned,
and values near the ends of their type."""

import importlib
import math
import threading

import pytest
import torch

import neural_shift_cuda_b200 as nsc
from neural_shift_cuda_b200 import _lib
from oracle import token_oracle as T
from token_cases import check, leaf, randn, reference

pytestmark = pytest.mark.gpu

A = importlib.import_module("neural_shift_cuda_b200.token_attention")

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


def _shifted(t):
    """t in storage that starts one element past an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.copy_(t.flatten()).view(t.shape)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 320])
def test_rotation_with_gradients_that_are_not_aligned(cuda, dt, D):
    """A contiguous gradient may start anywhere: a slice by the caller, or what the
    backward of a concatenation gives."""
    q, k = (randn(i, 2, 9, h, D, dtype=dt).to(cuda) for i, h in ((0, 4), (1, 2)))
    gq, gk = (randn(i, *t.shape, dtype=dt).to(cuda) for i, t in ((2, q), (3, k)))
    w = randn(4, D, dtype=dt).to(cuda)
    angle = torch.linspace(0, 3, 9 * D // 2, device=cuda).view(9, D // 2)
    cos, sin = angle.cos(), angle.sin()
    ref = [leaf(t.double()) for t in (q, k, w, w)]
    want = torch.autograd.grad(T.qk_norm_rotate(*ref, cos, sin), ref, [gq.double(), gk.double()])
    mine = [leaf(t) for t in (q, k, w, w)]
    out = nsc.qk_norm_rotate(*mine, cos, sin)
    one = torch.autograd.grad(out, mine, [_shifted(gq), _shifted(gk)], retain_graph=True)
    flat = torch.cat([q.new_zeros(1), out[0].flatten(), out[1].flatten()])
    two = torch.autograd.grad(flat, mine, torch.cat([q.new_zeros(1), gq.flatten(), gk.flatten()]))
    for got in (one, two):
        for g, x in zip(got, want):
            check(g, x, dt)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_rotation_to_outputs_that_are_not_aligned(cuda, dt):
    """The entry points take results and gradients at any address of their type."""
    q, k = (randn(i, 2, 9, h, 64, dtype=dt).to(cuda) for i, h in ((0, 4), (1, 2)))
    angle = torch.linspace(0, 3, 9 * 32, device=cuda).view(9, 32)
    a = A._rotate_args(q, k, None, None, angle.cos(), angle.sin(), None, 0, 1e-6)
    grads = [_shifted(k.repeat(1, 1, 2, 1)), _shifted(k)]
    for name, odd in (("nsc_qk_norm_rotate_fwd", []), ("nsc_qk_norm_rotate_bwd", grads)):
        tail = [None] * (3 if odd else 0)
        even = [t.clone() for t in odd]
        got, want = [_shifted(q), _shifted(k)], [torch.empty_like(q), torch.empty_like(k)]
        for ins, outs in ((odd, got), (even, want)):
            _lib.launch(q.device, name, a, *(t.data_ptr() for t in ins + outs), *tail)
        for x, y in zip(got, want):
            check(x, y, dt)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("L,D", [(40, 32), (200, 64), (200, 128)])
def test_attention_to_an_output_that_is_not_aligned(cuda, dt, L, D):
    """The entry points write out and residue at any address of their type."""
    q, k, v = (randn(i, 1, L, 2, D, dtype=dt).to(cuda) for i in range(3))
    want = T.attention(q, k, v, T.visible(1, L, L, True), D ** -0.5)[0]
    a = A._attention_args(q, k, v, None, None, None, None, None, D ** -0.5, 0.0, 1)
    for residue in (None, _shifted(q)):
        out = _shifted(q)
        _lib.launch(q.device, "nsc_token_attention_fwd", a, out.data_ptr(), None, None,
                    A._addr(residue))
        check(out, want, dt, "forward")
    n = torch.tensor([L], dtype=torch.int32, device=cuda)
    last = q[:, -1:]
    a = A._attention_args(last, k, v, None, None, n, None, None, D ** -0.5, 0.0, 1)
    ws = _lib.workspace("nsc_token_attention_decode_workspace", q.device, a)
    out = _shifted(last)
    _lib.launch(q.device, "nsc_token_attention_decode", a, out.data_ptr(), None, A._addr(ws))
    check(out, want[:, -1:], dt, "decode")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt,D", [(F16, 32), (BF16, 16), (BF16, 32), (F16, 8)])
@pytest.mark.parametrize("L,bounds", [(128, [0, 100]), (128, [28, 128]), (100, [0, 65]),
                                      (65, [1, 64]), (128, [70, 70]), (40, [5, 30])])
def test_short_rows_outside_all_documents(cuda, dt, D, L, bounds, causal):
    """Queries that see nothing, in tiles whose other queries all see a whole block of
    keys: out is 0 and lse -inf, and the gradients are those of the others."""
    q, k, v, go = (randn(i, 2, L, 4, D, dtype=dt).to(cuda) for i in range(4))
    m = nsc.relative_buckets(16, 40, device=cuda)
    table = randn(5, 16, 4, dtype=dt).to(cuda)
    rows = [bounds, [0, L]]
    doc = torch.tensor(rows, device=cuda)
    seen = T.visible(2, L, L, causal, None, rows)
    for tab, cap in ((None, 0.0), (table, 12.0)):
        kw = dict(documents=doc, causal=causal, softcap=cap, bias_table=tab,
                  bias_buckets=None if tab is None else m, return_lse=True)
        want = reference(q, k, v, seen, go, D ** -0.5, cap, tab, m)
        out, lse = nsc.token_attention(q, k, v, **kw)
        leaves = [leaf(t) for t in (q, k, v)]
        trained, lse2 = nsc.token_attention(*leaves, **kw)
        for o, x in ((out, lse), (trained, lse2)):
            check(o, want[0], dt, "out")
            check(x, want[1], F32, "lse", 8.0)
        for g, w in zip(torch.autograd.grad(trained, leaves, go), want[2:5]):
            check(g, w, dt)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("causal", [False, True])
def test_table_gradient_and_pairs_that_are_not_seen(cuda, dt, D, bad, cap, causal):
    """Output gradients of padding reach no bucket; those of a query that sees some keys
    reach the buckets of these and no other."""
    L, H = 300, 2
    q, k, v, go = (randn(i, 1, L, H, D, dtype=dt).to(cuda) for i in range(4))
    m = torch.arange(61, dtype=torch.int32, device=cuda)   # a bucket a distance, -30 .. 30
    doc = torch.tensor([[0, 140, 290]], device=cuda)

    def grad(go):
        t = leaf(randn(5, 61, H, dtype=dt).to(cuda))
        out = nsc.token_attention(q, k, v, documents=doc, causal=causal, softcap=cap,
                                  bias_table=t, bias_buckets=m)
        return torch.autograd.grad(out, t, go)[0]

    clean = grad(go)
    go2 = go.clone()
    go2[:, 290:] = bad
    assert torch.equal(grad(go2), clean)
    go2[:, 143] = bad     # sees keys 140 on: distances from -3
    got = grad(go2)
    last = 0 if causal else 30
    assert torch.equal(got[:27], clean[:27]) and torch.equal(got[30 + last + 1:],
                                                             clean[30 + last + 1:])
    assert not torch.isfinite(got[27:30 + last + 1]).any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("go_mul,lse_mul", [(1e-4, 1.0), (0.0, 2000.0), (1.0, 1e-3), (1.0, 30.0)])
@pytest.mark.parametrize("cap", [0.0, 10.0])
def test_fp16_gradients_of_lse(cuda, D, go_mul, lse_mul, cap):
    """Gradients of lse far above those of the output."""
    B, L, Hq, Hkv = 2, 300, 4, 2
    q = randn(0, B, L, Hq, D, dtype=F16).to(cuda)
    k, v = (randn(i, B, L, Hkv, D, dtype=F16).to(cuda) for i in (1, 2))
    go = randn(3, B, L, Hq, D, dtype=F16, mul=go_mul).to(cuda)
    gl = randn(4, B, Hq, L, dtype=F32, mul=lse_mul).to(cuda)
    doc = [[0, 7, 130, 290], [0, 1, 2, 300]]
    want = reference(q, k, v, T.visible(B, L, L, True, None, doc), go, D ** -0.5, cap, glse=gl)
    leaves = [leaf(t) for t in (q, k, v)]
    out, lse = nsc.token_attention(*leaves, causal=True, documents=torch.tensor(doc, device=cuda),
                                   softcap=cap, return_lse=True)
    got = torch.autograd.grad([out, lse], leaves, [go, gl])
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"), got, want[2:5]):
        check(g, w, F16, name)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("v_mul", [300.0, 4000.0])
def test_fp16_gradients_of_large_values(cuda, D, v_mul):
    """Value rows of norms in the thousands and more."""
    B, L, Hq, Hkv = 2, 333, 4, 2
    q = randn(0, B, L, Hq, D, dtype=F16).to(cuda)
    k = randn(1, B, L, Hkv, D, dtype=F16).to(cuda)
    v = randn(2, B, L, Hkv, D, dtype=F16, mul=v_mul).to(cuda)
    go = randn(3, B, L, Hq, D, dtype=F16).to(cuda)
    want = reference(q, k, v, T.visible(B, L, L, True), go, D ** -0.5)
    leaves = [leaf(t) for t in (q, k, v)]
    out = nsc.token_attention(*leaves, causal=True)
    got = torch.autograd.grad(out, leaves, go)
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"), got, want[2:5]):
        check(g, w, F16, name)


@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_beside_a_document_of_large_values(cuda, D):
    """The scale of one document's values and gradients is no matter of the others'."""
    L = 300
    q, k, v, go = (randn(i, 1, L, 2, D, dtype=F16).to(cuda) for i in range(4))
    doc = torch.tensor([[0, 140, 290]], device=cuda)
    leaves = [leaf(t) for t in (q, k, v)]
    ref = torch.autograd.grad(nsc.token_attention(*leaves, documents=doc), leaves, go)
    v2, go2 = v.clone(), go.clone()
    v2[:, 140:] *= 3000
    go2[:, 140:] *= 300
    leaves = [leaf(t) for t in (q, k, v2)]
    got = torch.autograd.grad(nsc.token_attention(*leaves, documents=doc), leaves, go2)
    for a, b in zip(got, ref):
        assert torch.equal(a[:, :140], b[:, :140])


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("cap", [200.0, 1e3, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("form", ["short", "decode"])
def test_large_caps_short_and_decode(cuda, dt, cap, form):
    """Scores far below the cap are as if there was none: their digits are their own, not
    those of the cap.  Prompt, short rows and cache agree."""
    Lq, Lk, D = (48, 48, 32) if form == "short" else (1, 400, 64)
    q = randn(0, 2, Lq, 4, D, dtype=dt, mul=2.0).to(cuda)
    k, v = (randn(i, 2, Lk, 2, D, dtype=dt, mul=2.0).to(cuda) for i in (1, 2))
    want, wl = T.attention(q, k, v, T.visible(2, Lq, Lk, True), D ** -0.5, cap)
    if form == "short":
        out, lse = nsc.token_attention(q, k, v, causal=True, softcap=cap, return_lse=True)
    else:
        n = torch.full((2,), Lk, dtype=torch.int32, device=cuda)
        out, lse = nsc.token_attention_decode(q, k, v, n, softcap=cap, return_lse=True)
    check(out, want, dt, "out")
    check(lse, wl, F32, "lse", 8.0)


@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 128), (F32, 64), (BF16, 32)])
@pytest.mark.parametrize("cap", [1e-3, 1e-5, 1e-8, 1e-12, 1e-20, 1e-30])
@pytest.mark.parametrize("L", [40, 300])
def test_small_caps(cuda, dt, D, cap, L):
    """Scores of zero stay zero, with a gradient, and all others are the cap's."""
    k, v, go = (randn(i, 1, L, 2, D, dtype=dt).to(cuda) for i in range(3))
    q = torch.zeros_like(k)
    want = reference(q, k, v, T.visible(1, L, L, True), go, D ** -0.5, cap)
    leaves = [leaf(t) for t in (q, k, v)]
    out = nsc.token_attention(*leaves, causal=True, softcap=cap)
    check(out, want[0], dt, "out")
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"),
                          torch.autograd.grad(out, leaves, go), want[2:5]):
        check(g, w, dt, name)
    q = randn(5, 1, L, 2, D, dtype=dt).to(cuda)
    leaves = [leaf(t) for t in (q, k, v)]
    want = reference(q, k, v, T.visible(1, L, L, True), go, D ** -0.5, cap)
    out = nsc.token_attention(*leaves, causal=True, softcap=cap)
    check(out, want[0], dt, "out")
    for g in torch.autograd.grad(out, leaves, go):
        assert torch.isfinite(g).all()
    n = torch.tensor([L], dtype=torch.int32, device=cuda)
    check(nsc.token_attention_decode(q[:, -1:], k, v, n, softcap=cap), want[0][:, -1:], dt)


@pytest.mark.parametrize("form,dt,D,less", [
    ("attention", F32, 96, 96), ("attention", F64, 64, 64), ("attention", BF16, 64, 64),
    ("decode", BF16, 72, 72), ("decode", F32, 130, 70), ("rotation", F64, 502, 300)])
def test_two_threads(cuda, form, dt, D, less):
    """Calls of one kernel that need more and less shared memory, from two threads."""
    def packed(width, bias):
        """The arguments of a small call, and what keeps them alive."""
        q = randn(0, 1, 3, 2, width, dtype=dt).to(cuda)
        out, dk = torch.empty_like(q), torch.empty_like(q)
        m = torch.zeros(2049, dtype=torch.int32, device=cuda)
        table = randn(1, 256, 2, dtype=dt).to(cuda)
        n = torch.tensor([3], dtype=torch.int32, device=cuda)
        if form == "rotation":
            angle = torch.zeros(3, width // 2, dtype=dt, device=cuda)
            a = A._rotate_args(q, q, None, None, angle, angle, None, 0, 1e-6)
            tail = (q, q, out, dk, None, None, None)
        else:
            a = A._attention_args(q, q, q, None, None, n if form == "decode" else None,
                                  table if bias else None, m if bias else None, 1.0, 0.0, 1)
            tail = (out, None, None, None) if form == "attention" else (out, None, None)
        return (a, *(A._addr(t) for t in tail)), (q, out, dk, m, table, n, a, tail)

    name = {"attention": "nsc_token_attention_fwd", "decode": "nsc_token_attention_decode",
            "rotation": "nsc_qk_norm_rotate_bwd"}[form]
    # (fewer channels, or no bias)
    calls = [packed(D, True), packed(less, False)]
    errors = []

    def work(args):
        with torch.cuda.stream(torch.cuda.Stream()):
            try:
                for i in range(4000):
                    _lib.launch(cuda_device, name, *args)
                    if i % 500 == 499:
                        torch.cuda.current_stream().synchronize()
            except RuntimeError as e:
                errors.append(e)

    cuda_device = calls[0][1][0].device
    for _ in range(3):
        ts = [threading.Thread(target=work, args=(c[0],)) for c in calls]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]


@pytest.mark.parametrize("dt", [F16, BF16, F32, F64])
@pytest.mark.parametrize("D", [32, 64])
def test_backward_of_an_empty_batch(cuda, dt, D):
    """Empty gradients, and zeros for the table."""
    m = nsc.relative_buckets(8, 20, device=cuda)
    for table in (None, torch.ones(8, 2, dtype=dt, device=cuda)):
        x = [torch.zeros(0, 70, 2, D, dtype=dt, device=cuda).requires_grad_() for _ in range(3)]
        t = leaf(table)
        out = nsc.token_attention(*x, bias_table=t, bias_buckets=None if t is None else m)
        got = torch.autograd.grad(out, x + ([t] if t is not None else []), torch.zeros_like(out))
        for g, w in zip(got, x):
            assert g.shape == w.shape
        if t is not None:
            assert (got[3] == 0).all()


def test_whole_numbers_past_32_bits(cuda):
    """int64 positions, lengths, bounds and prefixes are far away, not wrapped around."""
    big = 2 ** 32
    x = randn(0, 1, 3, 2, 64, dtype=BF16).to(cuda)
    angle = torch.linspace(0, 3, 8 * 32, device=cuda).view(8, 32)
    q, _ = nsc.qk_norm_rotate(x, x, None, None, angle.cos(), angle.sin(),
                              positions=torch.tensor([[0, big + 1, -big + 2]], device=cuda))
    assert torch.isfinite(q[:, 0]).all() and q[:, 1:].isnan().all()
    q, k, v = (randn(i, 1, 90, 2, 64, dtype=BF16).to(cuda) for i in range(3))
    for far in (big + 5, -big + 5):
        near = max(-2 ** 31, min(far, 2 ** 31 - 1))
        a = [nsc.token_attention_decode(q[:, :1], k, v, torch.tensor([n], device=cuda))
             for n in (far, near)]
        assert torch.equal(*a)
        a = [nsc.token_attention(q, k, v, documents=torch.tensor(sorted([7, n]), device=cuda))
             for n in (far, near)]
        assert torch.equal(*a)
        a = [nsc.token_attention(q, k, v, causal=True, prefix=torch.tensor([n], device=cuda))
             for n in (far, near)]
        assert torch.equal(*a)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F32, 64), (F64, 32)])
@pytest.mark.parametrize("scale", [0.0, -0.25])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_scales_of_zero_and_below(cuda, dt, D, scale, cap):
    """A scale of zero leaves the bias alone, with a cap or without."""
    q, k, v, go = (randn(i, 2, 90, 2, D, dtype=dt).to(cuda) for i in range(4))
    m = nsc.relative_buckets(16, 40, device=cuda)
    table = randn(5, 16, 2, dtype=dt).to(cuda)
    want = reference(q, k, v, T.visible(2, 90, 90, True), go, scale, cap, table, m)
    leaves = [leaf(t) for t in (q, k, v, table)]
    out = nsc.token_attention(*leaves[:3], scale=scale, softcap=cap, causal=True,
                              bias_table=leaves[3], bias_buckets=m)
    check(out, want[0], dt, "out")
    for name, g, w in zip(("grad_q", "grad_k", "grad_v", "grad_table"),
                          torch.autograd.grad(out, leaves, go), want[2:]):
        check(g, w, dt, name)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64)])
@pytest.mark.parametrize("wanted", ["q", "k", "v", "kv", "t", "qv", "qkv"])
def test_gradients_that_are_not_wanted(cuda, dt, D, wanted, monkeypatch):
    """Frozen inputs cost no kernel, and leave the others' gradients as they are."""
    q, k, v, go = (randn(i, 1, 300, 2, D, dtype=dt).to(cuda) for i in range(4))
    m = nsc.relative_buckets(16, 40, device=cuda)
    ins = dict(q=q, k=k, v=v, t=randn(5, 16, 2, dtype=dt).to(cuda))

    def run(names):
        x = {n: leaf(t) if n in names else t for n, t in ins.items()}
        out = nsc.token_attention(x["q"], x["k"], x["v"], causal=True, bias_table=x["t"],
                                  bias_buckets=m)
        return dict(zip(names, torch.autograd.grad(out, [x[n] for n in names], go)))

    want = run("qkvt")
    outputs = []
    pack = _lib.pack_attention_grad
    monkeypatch.setattr(_lib, "pack_attention_grad",
                        lambda *a: outputs.append(a[-5:-1]) or pack(*a))
    got = run(wanted)
    for n in wanted:
        assert torch.equal(got[n], want[n])
    dq, dk, dv, dt_ = (bool(x) for x in outputs[0])
    assert dt_ == ("t" in wanted) and dq == ("q" in wanted or dt_)
    assert dk == dv == ("k" in wanted or "v" in wanted)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (BF16, 40), (F64, 32)])
@pytest.mark.parametrize("wanted", [("q",), ("k",), ("wq",), ("wk",), ("q", "wk"), ("k", "wk")])
def test_rotation_gradients_that_are_not_wanted(cuda, dt, D, wanted, monkeypatch):
    ins = dict(q=randn(0, 2, 9, 4, D, dtype=dt).to(cuda), k=randn(1, 2, 9, 2, D, dtype=dt).to(cuda),
               wq=randn(2, D, dtype=dt).to(cuda), wk=randn(3, D, dtype=dt).to(cuda))
    angle = torch.linspace(0, 3, 9 * D // 2, device=cuda).view(9, D // 2)
    go = [randn(4, 2, 9, 4, D, dtype=dt).to(cuda), randn(5, 2, 9, 2, D, dtype=dt).to(cuda)]

    def run(names):
        x = {n: leaf(t) if n in names else t for n, t in ins.items()}
        out = nsc.qk_norm_rotate(*x.values(), angle.cos(), angle.sin())
        use = [i for i in (0, 1) if out[i].requires_grad]
        return dict(zip(names, torch.autograd.grad([out[i] for i in use], [x[n] for n in names],
                                                   [go[i] for i in use])))

    want = run(("q", "k", "wq", "wk"))
    outputs = []
    launch = _lib.launch
    monkeypatch.setattr(_lib, "launch", lambda *a: outputs.append(a) or launch(*a))
    got = run(wanted)
    for n in wanted:
        # (a weight's sum is over the blocks that its side has, which are more on its own)
        check(got[n], want[n], dt, n)
    dq, dk = (bool(x) for x in outputs[-1][5:7])
    assert dq == ("q" in wanted or "wq" in wanted) and dk == ("k" in wanted or "wk" in wanted)


@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("cap", [200.0, 500.0, 1e3, 1e4, 1e6, 1e30])
@pytest.mark.parametrize("mul", [2.0, 8.0])
def test_large_caps_tiles(cuda, dt, D, cap, mul):
    """Scores far below the cap.  The polynomial's slope at zero is short by 4.2e-5 (bf16),
    and lse, the largest score and little more, by as much: 16 times the usual bound of
    3.8e-6 leaves half as much again."""
    q, k, v, go = (randn(i, 1, 300, 2, D, dtype=dt, mul=mul if i < 2 else 1.0).to(cuda)
                   for i in range(4))
    want = reference(q, k, v, T.visible(1, 300, 300, True), go, D ** -0.5, cap)
    leaves = [leaf(t) for t in (q, k, v)]
    out, lse = nsc.token_attention(*leaves, causal=True, softcap=cap, return_lse=True)
    check(out, want[0], dt, "out")
    check(lse, want[1], F32, "lse", 16.0)
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"),
                          torch.autograd.grad(out, leaves, go), want[2:5]):
        check(g, w, dt, name)
