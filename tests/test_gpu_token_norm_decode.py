"""qk_norm_rotate and token_attention_decode against the 64-bit plain form."""

import math

import pytest
import torch

import neural_shift_cuda_b200 as nsc
from oracle import token_oracle as T
from token_cases import check, leaf, randn

pytestmark = pytest.mark.gpu

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


def _angles(rows, R, dt, dev):
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=F64) / max(R, 1))
    a = torch.arange(rows, dtype=F64)[:, None] * f
    acc = F64 if dt == F64 else F32
    return a.cos().to(dev, acc), a.sin().to(dev, acc)


def _rotate(dt, B, L, Hq, Hkv, D, R=None, adjacent=False, given=False, weights=True, seed=0,
            w_dt=None, view=None):
    dev = torch.device("cuda:0")
    R = D if R is None else R
    rows = L + 50 if given else L
    cos, sin = _angles(rows, R, dt, dev)
    pos = (torch.arange(B)[:, None] * 3 + torch.randperm(
        L, generator=torch.Generator().manual_seed(1))[None]).to(dev) % rows if given else None
    q = randn(seed, B, L, Hq, D, dtype=dt, mul=2.0).to(dev)
    k = randn(seed + 1, B, L, Hkv, D, dtype=dt, mul=0.3).to(dev)
    if view:
        q, k = view(q), view(k)
    wq = randn(seed + 2, D, dtype=w_dt or dt).to(dev) if weights else None
    wk = randn(seed + 3, D, dtype=w_dt or dt).to(dev) if weights else None
    gq = randn(seed + 4, B, L, Hq, D, dtype=dt).to(dev)
    gk = randn(seed + 5, B, L, Hkv, D, dtype=dt).to(dev)
    ref = [leaf(None if t is None else t.double()) for t in (q, k, wq, wk)]
    want = T.qk_norm_rotate(*ref, cos, sin, pos, adjacent)
    used = [t for t in ref if t is not None]
    wg = torch.autograd.grad(want, used, [gq.double(), gk.double()])
    mine = [leaf(t) for t in (q, k, wq, wk)]
    got = nsc.qk_norm_rotate(*mine, cos, sin, positions=pos, adjacent=adjacent)
    gg = torch.autograd.grad(got, [t for t in mine if t is not None], [gq, gk])
    for a, b in zip([*got, *gg], [*want, *wg]):
        check(a, b, dt if a.dtype == dt else F32, f"{a.shape}", 4.0 if a.dtype != dt else 1.0)
    with torch.no_grad():
        for a, b in zip(nsc.qk_norm_rotate(q, k, wq, wk, cos, sin, positions=pos,
                                           adjacent=adjacent), got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F16, BF16, F32, F64])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 96, 128, 256, 512])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotate_types_and_widths(cuda, dt, D, adjacent):
    _rotate(dt, 2, 17, 4, 2, D, adjacent=adjacent, given=adjacent)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("D", [8, 24, 40, 72, 136, 264, 272, 320])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotate_widths_of_eight(cuda, dt, D, adjacent):
    _rotate(dt, 2, 11, 5, 3, D, adjacent=adjacent, given=not adjacent)


@pytest.mark.parametrize("D,R", [(2, 2), (6, 4), (10, 10), (24, 8), (64, 32), (128, 0), (80, 48)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_rotate_odd_widths_and_part_of_the_channels(cuda, D, R, adjacent, dt):
    _rotate(dt, 2, 9, 3, 1, D, R, adjacent, given=True)


@pytest.mark.parametrize("B,L,Hq,Hkv", [(1, 1, 1, 1), (8, 1, 16, 4), (3, 257, 5, 5), (1, 2049, 12, 3),
                                        (2, 5, 40, 1), (0, 4, 2, 2), (2, 0, 2, 2)])
def test_rotate_extents(cuda, B, L, Hq, Hkv):
    if B * L:
        _rotate(BF16, B, L, Hq, Hkv, 64, given=True)
        return
    x = torch.zeros(B, L, 2, 64, dtype=BF16, device=cuda).requires_grad_()
    w = torch.ones(64, dtype=BF16, device=cuda).requires_grad_()
    cos, sin = _angles(8, 64, BF16, cuda)
    q, k = nsc.qk_norm_rotate(x, x, w, None, cos, sin)
    assert q.shape == x.shape
    assert (torch.autograd.grad(q.sum(), w)[0] == 0).all()


def test_rotate_without_weights_and_with_fp32_weights(cuda):
    _rotate(BF16, 2, 33, 4, 2, 128, weights=False)
    _rotate(F16, 2, 33, 4, 2, 128, w_dt=F32)
    _rotate(F16, 2, 33, 4, 2, 40, w_dt=F32)


@pytest.mark.parametrize("view", [
    lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
    lambda t: torch.cat([t, t], 2)[:, :, :t.shape[2]],
    lambda t: torch.nn.functional.pad(t, (1, 0))[..., 1:],
    lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)])
def test_rotate_strides(cuda, view):
    _rotate(BF16, 2, 19, 4, 2, 64, view=view)


def test_rotate_position_outside_the_table(cuda):
    x = randn(0, 1, 3, 2, 64, dtype=BF16).to(cuda)
    cos, sin = _angles(4, 64, BF16, cuda)
    for D in (64, 40):
        y = x[..., :D]
        q, k = nsc.qk_norm_rotate(y, y, None, None, cos[:, :D // 2], sin[:, :D // 2],
                                  positions=torch.tensor([[0, 4, -1]], device=cuda))
        assert torch.isfinite(q[:, 0]).all() and q[:, 1:].isnan().all() and k[:, 1:].isnan().all()


def test_rotate_against_differences(cuda):
    cos, sin = _angles(3, 4, F64, cuda)
    q = randn(0, 2, 3, 2, 6, dtype=F64).to(cuda).requires_grad_()
    k = randn(1, 2, 3, 1, 6, dtype=F64).to(cuda).requires_grad_()
    w = randn(2, 6, dtype=F64).to(cuda).requires_grad_()

    def f(q, k, w):
        return nsc.qk_norm_rotate(q, k, w, w, cos, sin)
    assert torch.autograd.gradcheck(f, (q, k, w), eps=1e-6, atol=1e-8, rtol=1e-6)


def test_rotate_zero_rows_and_same_bits(cuda):
    x = randn(0, 2, 300, 6, 64, dtype=BF16).to(cuda)
    x[:, 5] = 0
    cos, sin = _angles(300, 64, BF16, cuda)

    def once():
        a, w = leaf(x), leaf(torch.ones(64, device=cuda, dtype=BF16))
        q, k = nsc.qk_norm_rotate(a, a, w, w, cos, sin)
        return q, k, *torch.autograd.grad((q.float() * k.float()).sum(), [a, w])
    first, second = once(), once()
    assert (first[0][:, 5] == 0).all()
    for a, b in zip(first, second):
        assert torch.isfinite(a).all() and torch.equal(a, b)


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------

def _decode(dt, lengths, T_new, Hq, Hkv, D, cap=0.0, buckets=None, extra=7, seed=0, garbage=None):
    dev = torch.device("cuda:0")
    B, n = len(lengths), max(max(lengths) + extra, 1)
    q = randn(seed, B, T_new, Hq, D, dtype=dt, mul=1.3).to(dev)
    k = randn(seed + 1, B, n, Hkv, D, dtype=dt, mul=1.3).to(dev)
    v = randn(seed + 2, B, n, Hkv, D, dtype=dt).to(dev)
    if garbage is not None:
        for b, m in enumerate(lengths):
            k[b, m:] = garbage
            v[b, m:] = garbage
    m = t = None
    if buckets:
        m = nsc.relative_buckets(*buckets, device=dev)
        t = randn(seed + 3, buckets[0], Hq, dtype=dt).to(dev)
    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    got, lse = nsc.token_attention_decode(q, k, v, ln, softcap=cap, bias_table=t, bias_buckets=m,
                                          return_lse=True)
    seen = T.visible(B, T_new, n, True, lengths=lengths)
    for b, m_ in enumerate(lengths):
        k[b, m_:] = 0
        v[b, m_:] = 0
    want, wl = T.attention(q, k, v, seen, D ** -0.5, cap, t, m,
                           offset=torch.tensor(lengths) - T_new)
    check(got, want, dt, "out")
    check(lse, wl, F64 if dt == F64 else F32, "lse", 8.0)
    again = nsc.token_attention_decode(
        q, k, v, ln, softcap=cap, bias_table=t, bias_buckets=m)
    assert torch.equal(again, got)


@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 128), (F32, 64), (F64, 32), (BF16, 32),
                                  (F16, 96), (BF16, 256), (F32, 128), (BF16, 40), (F16, 7)])
@pytest.mark.parametrize("T_new", [1, 4])
def test_decode_types_and_widths(cuda, dt, D, T_new):
    _decode(dt, [1, 37, 200, 513], T_new, 8, 2, D)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (16, 16), (5, 1), (16, 1), (24, 3), (40, 2), (64, 1)])
@pytest.mark.parametrize("T_new", [1, 2, 5, 8])
def test_decode_head_groups(cuda, Hq, Hkv, T_new):
    _decode(BF16, [130, 64], T_new, Hq, Hkv, 64)


@pytest.mark.parametrize("lengths", [[0], [0, 0, 5], [1], [2, 63, 64, 65], [127, 128, 129],
                                     [3000, 1, 0, 17], [9001]])
@pytest.mark.parametrize("T_new", [1, 3])
def test_decode_lengths(cuda, lengths, T_new):
    _decode(BF16, lengths, T_new, 4, 2, 64, garbage=math.nan)
    _decode(F32, lengths, T_new, 4, 2, 64, garbage=math.inf)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_decode_cap_and_bias(cuda, dt, D):
    _decode(dt, [700, 33, 1500], 1, 8, 2, D, cap=6.0)
    _decode(dt, [700, 33, 1500], 4, 8, 2, D, buckets=(32, 128, True))
    _decode(dt, [700, 33, 1500], 3, 8, 2, D, cap=8.0, buckets=(16, 300, False))


def test_decode_many_new_tokens(cuda):
    _decode(BF16, [300, 40], 40, 8, 2, 64, cap=9.0)
    _decode(BF16, [300, 40], 70, 4, 4, 128)


def test_decode_strides(cuda):
    """Head-major caches, a layer's slice of a shared cache, unaligned rows."""
    for dt, D in ((BF16, 64), (F32, 64)):
        q = randn(0, 2, 1, 8, D, dtype=dt).to(cuda)
        k = randn(1, 2, 300, 2, D, dtype=dt).to(cuda)
        v = randn(2, 2, 300, 2, D, dtype=dt).to(cuda)
        ln = torch.tensor([300, 211], device=cuda)
        want = nsc.token_attention_decode(q, k, v, ln)
        hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
        assert torch.equal(nsc.token_attention_decode(q, *hm, ln), want)
        both = torch.stack([k, v], 2)
        assert torch.equal(nsc.token_attention_decode(q, both[:, :, 0], both[:, :, 1], ln), want)
        odd = [torch.nn.functional.pad(t, (1, 0))[..., 1:] for t in (k, v)]
        check(nsc.token_attention_decode(q, *odd, ln), want, dt)


def test_decode_offsets_past_32_bits(cuda):
    """The last sequence of a cache of more than 2^32 elements."""
    rows, D = 4200000, 64
    k = torch.zeros(16, rows, 1, D, dtype=F16, device=cuda)
    tail = randn(1, 300, 1, D, dtype=F16).to(cuda)
    k[15, :300] = tail
    q = randn(2, 16, 1, 2, D, dtype=F16).to(cuda)
    ln = torch.full((16,), 300, dtype=torch.int32, device=cuda)
    got = nsc.token_attention_decode(q, k, k, ln)
    # (the cut of the long axis goes by the cache's rows, so not bit for bit)
    want = T.attention(q[15:], tail[None], tail[None], T.visible(1, 1, 300), D ** -0.5)[0]
    check(got[15:], want, F16)


def test_decode_agrees_with_attention(cuda):
    """A prompt through token_attention, token by token through the cache."""
    q, k, v = (randn(i, 1, 150, 4, 64, dtype=F32).to(cuda) for i in range(3))
    whole = nsc.token_attention(q, k, v, causal=True, softcap=5.0)
    for n in (1, 2, 77, 150):
        one = nsc.token_attention_decode(q[:, n - 1:n], k, v, torch.tensor([n], device=cuda),
                                         softcap=5.0)
        check(one, whole[:, n - 1:n], F32)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_a_layer_in_a_graph(cuda, dt):
    """Prompt, few new queries and decode, captured once and replayed on new values."""
    B, n, H, Hk, D = 2, 300, 4, 2, 64
    x = randn(0, B, n, H + 2 * Hk, D, dtype=dt).to(cuda)
    cos, sin = _angles(n, D, dt, cuda)
    lengths = torch.tensor([n, 211], dtype=torch.int32, device=cuda)

    def layer():
        q, k, v = x.split((H, Hk, Hk), 2)
        q, k = nsc.qk_norm_rotate(q, k, None, None, cos, sin)
        return (nsc.token_attention(q, k, v, causal=True, softcap=9.0),
                nsc.token_attention(q[:, -2:], k, v, causal=True),
                nsc.token_attention_decode(q[:, -3:], k, v, lengths))

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer()
        for seed in (1, 2):
            x.copy_(randn(seed, *x.shape, dtype=dt))
            graph.replay()
            for a, b in zip(got, layer()):
                assert torch.equal(a, b)
