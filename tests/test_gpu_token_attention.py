"""Token attention against the 64-bit plain form: types, head layouts, lengths
from none to long, masks, caps, biases, and every gradient."""

import math

import pytest
import torch

import neural_shift_cuda_b200 as nsc
from oracle import token_oracle as T
from token_cases import U, check, leaf, randn, reference

pytestmark = pytest.mark.gpu

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


def _mask(B, Lq, Lk, kind, dev):
    """(kwargs of token_attention, visible pairs)"""
    if kind == "full":
        return {}, T.visible(B, Lq, Lk)
    if kind == "causal":
        return {"causal": True}, T.visible(B, Lq, Lk, True)
    if kind == "prefix":
        pre = torch.tensor([(7 * b + Lk // 3) % (Lk + 1) for b in range(B)])
        return ({"causal": True, "prefix": pre.to(dev)},
                T.visible(B, Lq, Lk, True, pre[:, None]))
    # documents of uneven length, an empty one, padding after the last
    rows = []
    for b in range(B):
        a, c, e = Lk // 5, (Lk * 3) // 5 + b % 2, Lk - Lk // 11
        rows.append([0, a, a, max(a, c), max(a, c, e)])
    doc = torch.tensor(rows)
    if kind == "docs":
        return {"documents": doc.to(dev)}, T.visible(B, Lq, Lk, False, None, rows)
    if kind == "docs_causal":
        return ({"documents": doc.to(dev, torch.int32), "causal": True},
                T.visible(B, Lq, Lk, True, None, rows))
    pre = torch.tensor([[2, 3, 5, 1 + 9 * b] for b in range(B)])
    return ({"documents": doc.to(dev), "causal": True, "prefix": pre.to(dev)},
            T.visible(B, Lq, Lk, True, pre, rows))


def _run(dt, B, Lq, Lk, Hq, Hkv, D, kind, cap=0.0, buckets=None, mul=1.0, seed=0, glse=False,
         table_dt=None):
    dev = torch.device("cuda:0")
    q = randn(seed, B, Lq, Hq, D, dtype=dt, mul=mul).to(dev)
    k = randn(seed + 1, B, Lk, Hkv, D, dtype=dt, mul=mul).to(dev)
    v = randn(seed + 2, B, Lk, Hkv, D, dtype=dt).to(dev)
    go = randn(seed + 3, B, Lq, Hq, D, dtype=dt).to(dev)
    gl = randn(seed + 4, B, Hq, Lq, dtype=F64 if dt == F64 else F32).to(dev) if glse else None
    table = m = None
    if buckets:
        m = nsc.relative_buckets(*buckets, device=dev)
        table = randn(seed + 5, buckets[0], Hq, dtype=table_dt or dt).to(dev)
    kw, seen = _mask(B, Lq, Lk, kind, dev)
    scale = D ** -0.5
    want = reference(q, k, v, seen, go, scale, cap, table, m, gl)
    ql, kl, vl, tl = leaf(q), leaf(k), leaf(v), leaf(table)
    out, lse = nsc.token_attention(ql, kl, vl, softcap=cap, bias_table=tl, bias_buckets=m,
                                   return_lse=True, **kw)
    loss = (out * go).sum() if gl is None else None
    ins = [ql, kl, vl] + ([tl] if tl is not None else [])
    if gl is None:
        got = torch.autograd.grad(out, ins, go)
    else:
        got = torch.autograd.grad([out, lse], ins, [go, gl])
    del loss
    check(out, want[0], dt, "out")
    check(lse, want[1], F64 if dt == F64 else F32, "lse", 8.0)
    for name, g, w in zip(("grad_q", "grad_k", "grad_v"), got, want[2:5]):
        check(g, w, dt, name)
    if table is not None:
        # score gradients of both signs cancel in a bucket's sum; its error is
        # that of the softmax statistics, not of the table's type
        check(got[3], want[5], dt, "grad_table")
    with torch.no_grad():
        again = nsc.token_attention(q, k, v, softcap=cap, bias_table=table, bias_buckets=m, **kw)
    if dt in (F32, F64):
        assert torch.equal(again, out.detach())
    else:   # training keeps more digits of the weights
        check(again, want[0], dt, "out without gradients")
    return out, got


@pytest.mark.parametrize("kind", ["full", "causal", "prefix", "docs", "docs_causal",
                                  "docs_prefix"])
@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 128), (F32, 64), (F64, 32)])
def test_masks(cuda, kind, dt, D):
    _run(dt, 2, 203, 203, 4, 2, D, kind)


@pytest.mark.parametrize("Lq,Lk", [(1, 40), (2, 129), (63, 64), (127, 128), (128, 128),
                                   (129, 127), (130, 257), (255, 256), (257, 300), (300, 130),
                                   (385, 513)])
@pytest.mark.parametrize("kind", ["full", "causal", "prefix"])
def test_lengths(cuda, Lq, Lk, kind):
    _run(BF16, 1, Lq, Lk, 2, 1, 64, kind, seed=Lq)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64), (F64, 32)])
def test_one_token(cuda, dt, D):
    """One key: out = v, grad_v = grad_out, and the gradients of q and k are
    zero, as differences of two sums of D products: each is within 2 u of the
    sum of their magnitudes, of which q.k's factor takes its share."""
    q, k, v, go = (randn(i, 1, 1, 2, D, dtype=dt).to(cuda) for i in range(4))
    leaves = [leaf(t) for t in (q, k, v)]
    out = nsc.token_attention(*leaves, causal=True)
    dq, dk, dv = torch.autograd.grad(out, leaves, go)
    assert torch.equal(out, v) and torch.equal(dv, go)
    dz = 2 * U[F64 if dt == F64 else F32] * (go * v).double().abs().sum(-1, keepdim=True) * D ** 0.5
    assert (dq.double().abs() <= dz * k.double().abs() * D ** -0.5).all()
    assert (dk.double().abs() <= dz * q.double().abs() * D ** -0.5).all()


@pytest.mark.parametrize("D", [1, 5, 8, 16, 24, 32, 40, 72, 80, 96, 112, 128, 136, 200, 256])
def test_head_widths(cuda, D):
    _run(F16, 1, 75, 140, 2, 2, D, "causal", seed=D)


@pytest.mark.parametrize("D", [3, 64, 100, 192])
def test_head_widths_f32(cuda, D):
    _run(F32, 1, 75, 70, 2, 2, D, "causal", seed=D)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (8, 1), (6, 3), (8, 8), (12, 2)])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_shared_heads(cuda, Hq, Hkv, dt):
    _run(dt, 3, 140, 140, Hq, Hkv, 64, "docs_causal")


@pytest.mark.parametrize("dt,D,cap,mul", [(BF16, 64, 5.0, 1.5), (F16, 128, 30.0, 2.0),
                                          (BF16, 128, 2.0, 3.0), (F32, 64, 4.0, 2.0),
                                          (F64, 16, 3.0, 2.0)])
@pytest.mark.parametrize("kind", ["full", "docs_prefix"])
def test_softcap(cuda, dt, D, cap, mul, kind):
    _run(dt, 2, 150, 150, 4, 2, D, kind, cap, mul=mul)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64), (F64, 32)])
@pytest.mark.parametrize("buckets", [(8, 20, True), (32, 128, True), (16, 9, False),
                                     (64, 700, True)])
def test_bias(cuda, dt, D, buckets):
    _run(dt, 2, 290, 290, 4, 2, D, "full", buckets=buckets)


@pytest.mark.parametrize("kind,cap,Lq,Lk", [("causal", 6.0, 200, 333), ("prefix", 0.0, 130, 129),
                                            ("docs_prefix", 8.0, 260, 260)])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_bias_with_masks(cuda, kind, cap, Lq, Lk, dt):
    _run(dt, 2, Lq, Lk, 6, 2, 64, kind, cap, buckets=(32, 64, True), mul=1.5)


def test_bias_table_in_fp32(cuda):
    _run(BF16, 2, 150, 150, 4, 4, 64, "causal", buckets=(8, 20, True), table_dt=F32)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F32, 32), (F64, 32)])
def test_lse_gradient(cuda, dt, D):
    _run(dt, 2, 140, 140, 4, 2, D, "causal", glse=True)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (BF16, 128)])
def test_long(cuda, dt, D):
    _run(dt, 1, 2085, 2085, 2, 1, D, "docs_prefix", 20.0, buckets=(32, 128, True), mul=1.5)
    _run(dt, 1, 1500, 2700, 2, 2, D, "full", mul=1.5)


def test_large_scores_move_the_reference(cuda):
    """Scores that grow along the row by hundreds: the running maximum moves
    many times, far past the range of an unscaled exponential."""
    dev = cuda
    for dt, D in ((BF16, 64), (BF16, 128), (F32, 64)):
        q = randn(1, 1, 140, 2, D, dtype=dt).to(dev)
        k = randn(2, 1, 900, 2, D, dtype=dt).to(dev)
        ramp = torch.linspace(0.1, 12.0, 900, device=dev)[None, :, None, None]
        k = (k.float() * ramp).to(dt)
        v = randn(3, 1, 900, 2, D, dtype=dt).to(dev)
        want, lse = T.attention(q, k, v, T.visible(1, 140, 900), 0.5)
        got, gl = nsc.token_attention(q, k, v, scale=0.5, return_lse=True)
        check(got, want, dt, "out", 4.0)
        check(gl, lse, F32, "lse", 8.0)


def test_softcap_at_large_scores(cuda):
    for dt, D in ((F16, 64), (BF16, 128), (F32, 32)):
        _run(dt, 1, 140, 260, 2, 1, D, "causal", cap=10.0, mul=6.0)


@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 128), (F32, 64)])
def test_strides_and_order(cuda, dt, D):
    """Slices of one projection, head-major storage, a reversed batch order by
    index, and rows whose stride is not a multiple of 16 bytes."""
    x = randn(5, 2, 170, 8, D, dtype=dt).to(cuda)
    q, k, v = x[:, :, :4], x[:, :, 4:6], x[:, :, 6:]
    want = nsc.token_attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(nsc.token_attention(q, k, v, causal=True), want)
    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(nsc.token_attention(*hm, causal=True), want)
    odd = torch.empty(2, 170, 8 * D + 1, dtype=dt, device=cuda)
    odd = odd[:, :, 1:].unflatten(-1, (8, D))
    odd.copy_(x)
    seen = T.visible(2, 170, 170, True)
    go = randn(6, 2, 170, 4, D, dtype=dt).to(cuda)
    ref = reference(q, k, v, seen, go, D ** -0.5)
    leaves = [leaf(odd[:, :, a:b]) for a, b in ((0, 4), (4, 6), (6, 8))]
    out = nsc.token_attention(*leaves, causal=True)
    check(out, ref[0], dt)
    for g, w in zip(torch.autograd.grad(out, leaves, go.transpose(1, 2).contiguous()
                                        .transpose(1, 2)), ref[2:5]):
        check(g, w, dt)
    # a broadcast key head and a last dimension that is not unit stride
    one = x[:, :, 4:5].expand(2, 170, 4, D)
    check(nsc.token_attention(q, one, one),
          T.attention(q, one, one, T.visible(2, 170, 170), D ** -0.5)[0], dt)
    tr = x.transpose(-1, -2).contiguous().transpose(-1, -2)
    check(nsc.token_attention(tr[:, :, :4], tr[:, :, 4:6], tr[:, :, 6:], causal=True), ref[0], dt)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_seen_has_no_influence(cuda, dt, D, bad):
    """NaN and infinities in keys, values, queries and output gradients of one
    document leave the other documents' results and gradients as they are;
    so do those in padding, and in a causal row's future."""
    L = 300
    q, k, v, go = (randn(i, 1, L, 2, D, dtype=dt).to(cuda) for i in range(4))
    doc = torch.tensor([[0, 140, 290]], device=cuda)
    kw = dict(documents=doc, causal=True)
    leaves = [leaf(t) for t in (q, k, v)]
    out = nsc.token_attention(*leaves, **kw)
    ref = torch.autograd.grad(out, leaves, go)
    q2, k2, v2, go2 = (t.clone() for t in (q, k, v, go))
    for t in (q2, k2, v2, go2):
        t[:, 290:] = bad        # padding
        t[:, 200:210] = bad     # tokens of the second document
    leaves2 = [leaf(t) for t in (q2, k2, v2)]
    out2 = nsc.token_attention(*leaves2, **kw)
    got = torch.autograd.grad(out2, leaves2, go2)
    assert torch.equal(out2[:, :200], out[:, :200])
    assert (out2[:, 290:] == 0).all() and not torch.isfinite(out2[:, 200:290]).all()
    for a, b in zip(got, ref):
        assert torch.equal(a[:, :140], b[:, :140])
        assert (a[:, 290:] == 0).all()


@pytest.mark.parametrize("dt,D", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("mul", [2.0 ** -12, 1.0, 2.0 ** 8])
def test_scale_of_the_output_gradient(cuda, dt, D, mul):
    """Long uniform rows and small (or large) output gradients: weights and
    score gradients far below the normal range of fp16, or near its end.
    Powers of two scale the gradients and nothing else; what fp16 cannot
    hold of them (below 2^-24) bounds the rest."""
    q, k, v, go = (randn(i, 1, 1200, 2, D, dtype=dt, mul=m).to(cuda)
                   for i, m in ((0, 0.3), (1, 0.3), (2, 1.0), (3, 1.0)))
    go = go * mul
    leaves = [leaf(t) for t in (q, k, v)]
    got = torch.autograd.grad(nsc.token_attention(*leaves), leaves, go)
    want = reference(q, k, v, T.visible(1, 1200, 1200), go, D ** -0.5)[2:5]
    floor = 2.0 ** -24 if dt == F16 else 0.0
    for g, w in zip(got, want):
        d = (g.double() - w).norm()
        assert d <= 3 * U[dt] * w.norm() + floor * w.numel() ** 0.5


def test_rows_that_see_nothing(cuda):
    for dt in (BF16, F32):
        q, k, v = (randn(i, 2, 200, 2, 64, dtype=dt).to(cuda) for i in range(3))
        leaves = [leaf(t) for t in (q, k, v)]
        doc = torch.tensor([[0, 0], [150, 150]], device=cuda)
        out, lse = nsc.token_attention(*leaves, documents=doc, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
        for g in torch.autograd.grad(out, leaves, torch.ones_like(out)):
            assert (g == 0).all()
        # the first queries of a chunk that is longer than its keys
        out, lse = nsc.token_attention(q, k[:, :130], v[:, :130], causal=True, return_lse=True)
        assert (out[:, :70] == 0).all() and (lse[:, :, :70] == -math.inf).all()
        assert torch.isfinite(lse[:, :, 70:]).all()


def test_bias_of_the_lowest_value_and_of_minus_infinity(cuda):
    """A bucket at the type's lowest value hides its pairs behind any other,
    and leaves a uniform softmax where a row has nothing else; a bucket of
    -inf hides them for good."""
    for dt, D in ((BF16, 64), (F16, 128), (F32, 64)):
        q, k, v = (randn(i, 1, 150, 1, D, dtype=dt).to(cuda) for i in range(3))
        m = torch.zeros(21, dtype=torch.int32, device=cuda)
        m[:10] = 1
        for low in (torch.finfo(dt).min, -math.inf):
            table = torch.tensor([[0.0], [low]], dtype=dt, device=cuda)
            want, lse = T.attention(q, k, v, T.visible(1, 150, 150), 0.125, 0.0, table, m)
            leaves = [leaf(q), leaf(k), leaf(v), leaf(table)]
            got = nsc.token_attention(*leaves[:3], scale=0.125, bias_table=leaves[3],
                                      bias_buckets=m)
            check(got, want, dt)
            for g in torch.autograd.grad(got, leaves, torch.ones_like(got)):
                assert torch.isfinite(g).all()
        # only far-past keys of that bucket are left to the last queries
        table = torch.tensor([[0.0], [-math.inf]], dtype=dt, device=cuda)
        out, lse = nsc.token_attention(q[:, 100:], k[:, :50], v[:, :50], scale=0.125,
                                       bias_table=table,
                                       bias_buckets=torch.ones_like(m), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_nan_in_a_seen_place_shows(cuda):
    for dt, D in ((BF16, 64), (F32, 64)):
        q, k, v = (randn(i, 1, 200, 1, D, dtype=dt).to(cuda) for i in range(3))
        k[:, 60] = math.nan
        out = nsc.token_attention(q, k, v, causal=True)
        assert torch.isfinite(out[:, :60]).all() and out[:, 60:].isnan().all()


def test_same_bits_again_and_on_another_stream(cuda):
    for dt, D in ((BF16, 128), (F32, 64)):
        q, k, v, go = (randn(i, 2, 400, 4, D, dtype=dt).to(cuda) for i in range(4))
        m = nsc.relative_buckets(16, 40, device=cuda)
        t = randn(7, 16, 4, dtype=dt).to(cuda)

        def once():
            leaves = [leaf(x) for x in (q, k, v, t)]
            out = nsc.token_attention(*leaves[:3], causal=True, bias_table=leaves[3],
                                      bias_buckets=m)
            return [out, *torch.autograd.grad(out, leaves, go)]
        first = once()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = once()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a, b in zip(first, second):
            assert torch.equal(a, b)


def test_gradients_against_differences(cuda):
    q, k, v = (randn(i, 1, 6, 2, 4, dtype=F64).to(cuda).requires_grad_() for i in range(3))
    m = nsc.relative_buckets(8, 5, device=cuda)
    t = randn(4, 8, 2, dtype=F64).to(cuda).requires_grad_()
    doc = torch.tensor([0, 4, 6], device=cuda)

    def f(q, k, v, t):
        return nsc.token_attention(q, k, v, softcap=2.0, causal=True, prefix=2, documents=doc,
                                   bias_table=t, bias_buckets=m, return_lse=True)
    assert torch.autograd.gradcheck(f, (q, k, v, t), eps=1e-6, atol=1e-8, rtol=1e-6)


def test_no_queries_or_no_keys(cuda):
    z = torch.zeros(2, 0, 2, 64, dtype=BF16, device=cuda)
    x = randn(1, 2, 9, 2, 64, dtype=BF16).to(cuda)
    assert nsc.token_attention(z, x, x).shape == (2, 0, 2, 64)
    out, lse = nsc.token_attention(x, z, z, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    leaves = [leaf(x), leaf(z), leaf(z)]
    for g in torch.autograd.grad(nsc.token_attention(*leaves), leaves, x):
        assert (g == 0).all()
    leaves = [leaf(z), leaf(x), leaf(x)]
    for g in torch.autograd.grad(nsc.token_attention(*leaves), leaves, z):
        assert (g == 0).all()
    e = torch.zeros(0, 5, 2, 64, dtype=BF16, device=cuda)
    assert nsc.token_attention(e, e, e).shape == (0, 5, 2, 64)


def test_slow_and_fast_warps_keep_in_step(cuda):
    """Warps whose scores pass the cap's polynomial take far longer than others; no
    block of products may start before the slowest has written its part."""
    for dt, D in ((BF16, 64), (F16, 64), (BF16, 128)):
        q = randn(0, 1, 140, 2, D, dtype=dt, mul=6.0).to(cuda)
        k = randn(1, 1, 700, 1, D, dtype=dt, mul=6.0).to(cuda)
        k[:, ::3] *= 0.01
        v = randn(2, 1, 700, 1, D, dtype=dt).to(cuda)
        go = randn(3, 1, 140, 2, D, dtype=dt).to(cuda)
        first = None
        for _ in range(12):
            leaves = [leaf(t) for t in (q, k, v)]
            out = nsc.token_attention(*leaves, causal=True, softcap=10.0)
            now = [out, *torch.autograd.grad(out, leaves, go)]
            first = first or now
            for a, b in zip(first, now):
                assert torch.equal(a, b)


@pytest.mark.parametrize("L", [96, 387])
@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 64), (BF16, 128)])
def test_score_gradients_of_rows_with_few_keys(cuda, dt, D, L):
    """Documents of three tokens: a score's gradient is a small difference, of the
    weights' gradients and the row's sum of grad_out * out.  What reaches grad_q and
    grad_k is their own rounding; a quarter more is left for all else."""
    q, k, v, go = (randn(71 + i, 2, L, 4, D, dtype=dt, mul=1.5 if i < 2 else 1.0).to(cuda)
                   for i in range(4))
    rows = [list(range(0, L + 1, 3))] * 2
    want = reference(q, k, v, T.visible(2, L, L, False, None, rows), go, D ** -0.5)
    ql, kl, vl = leaf(q), leaf(k), leaf(v)
    out = nsc.token_attention(ql, kl, vl, documents=torch.tensor(rows, device=cuda))
    got = torch.autograd.grad(out, [ql, kl, vl], go)
    for name, g, w in zip(("grad_q", "grad_k"), got, want[2:4]):
        own = float((w.to(dt).double() - w).norm() / w.norm())
        off = float((g.double() - w).norm() / w.norm())
        print(name, own, off)
        assert off <= 1.25 * own, f"{name}: {off:.3g}, its own rounding is {own:.3g}"


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt,D,Lq,Lk,Hq,Hkv", [
    (BF16, 64, 1, 256, 4, 4), (BF16, 128, 4, 300, 8, 2), (F16, 64, 16, 700, 2, 2),
    (BF16, 128, 5, 2100, 12, 2), (F16, 96, 64, 2048, 4, 1), (BF16, 40, 33, 4097, 2, 1),
    (F32, 64, 1, 1000, 4, 2), (F32, 128, 16, 259, 3, 1), (F32, 36, 7, 513, 8, 1)])
def test_few_queries_over_many_keys(cuda, dt, D, Lq, Lk, Hq, Hkv, causal):
    """Without gradients such a call shares out the keys over the GPU."""
    for cap, buckets in ((0.0, None), (7.0, (16, 60, True) if causal else None)):
        q = randn(1, 2, Lq, Hq, D, dtype=dt).to(cuda)
        k = randn(2, 2, Lk, Hkv, D, dtype=dt).to(cuda)
        v = randn(3, 2, Lk, Hkv, D, dtype=dt).to(cuda)
        table = m = None
        if buckets:
            m = nsc.relative_buckets(*buckets, device=cuda)
            table = randn(4, buckets[0], Hq, dtype=dt).to(cuda)
        seen = T.visible(2, Lq, Lk, causal)
        want, lse = T.attention(q, k, v, seen, D ** -0.5, cap, table, m)
        got, gl = nsc.token_attention(q, k, v, causal=causal, softcap=cap, bias_table=table,
                                      bias_buckets=m, return_lse=True)
        check(got, want, dt, "out")
        check(gl, lse, F32, "lse", 8.0)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F32, 64)])
def test_few_queries_and_values_that_are_not_finite(cuda, dt, D):
    """A key past a query has no influence; where a key is seen it has."""
    q, k, v = (randn(i, 1, 3 if i == 0 else 400, 2, D, dtype=dt).to(cuda) for i in range(3))
    want = nsc.token_attention(q, k, v, causal=True)
    v2, k2 = v.clone(), k.clone()
    v2[:, 398:] = math.inf
    k2[:, 399:] = math.nan
    got = nsc.token_attention(q, k2, v2, causal=True)
    assert torch.equal(got[:, 0], want[:, 0])
    assert not torch.isfinite(got[:, 1:]).any()
    every = nsc.token_attention(q, k2, v2)
    assert not torch.isfinite(every).any()
