"""Token attention on B200: the operators of the transformer layers that run
beside the shift-window denoisers (token mixers over image patches, image
language models, diffusion transformers).

    qk_norm_rotate(q, k, q_weight, k_weight, cos, sin)      -> (q', k')
    token_attention(q, k, v, ...)                           -> out
    token_attention_decode(q, k_cache, v_cache, lengths)    -> out
    relative_buckets(num_buckets, max_distance)             -> bucket map

Where `normalized_accumulate_uz` is a softmax over a fixed window of shifts
with given logits, `token_attention` is the softmax over all tokens whose
logits are products of queries and keys, capped by a tanh, with a learned
bias by buckets of distance, under causal, prefix and document masks.
Tensors are (B, L, H, D) with any strides of B, L and H, so the slices of one
projection are read in place; fp16, bf16, fp32 and fp64; sums and softmax
statistics in fp32 (fp64).  CUDA tensors only, as the other ops.  Nothing here
has a counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["qk_norm_rotate", "token_attention", "token_attention_decode",
           "relative_buckets"]


# ---------------------------------------------------------------------------
# argument handling
# ---------------------------------------------------------------------------

def _require_cuda(op: str, q: torch.Tensor) -> None:
    """(The other tensors are known to share q's device.)"""
    if not q.is_cuda:
        raise RuntimeError(
            f"neural_shift_cuda_b200.{op}: expects CUDA tensors (got a "
            f"{q.device} tensor); this package has no CPU path")
    _lib.load()


def _refuse_tangents(op: str, *tensors: Optional[torch.Tensor]) -> None:
    """A call that records no graph passes by the autograd functions, which would refuse
    tangents: they would be dropped."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{op} has no forward-mode derivative")


def _check_heads(op: str, name: str, t: torch.Tensor) -> None:
    if t.ndim != 4:
        raise RuntimeError(f"{op}: {name} must be (B, L, H, D); got "
                           f"{tuple(t.shape)}")


def _check_like(op: str, q: torch.Tensor, **others: torch.Tensor) -> None:
    if q.dtype not in _lib._DTYPES:
        raise TypeError(f"{op}: unsupported dtype {q.dtype}")
    for name, t in others.items():
        if t.dtype != q.dtype:
            raise TypeError(f"{op}: {name} is {t.dtype}, q is {q.dtype}")
        if t.device != q.device:
            raise ValueError(f"{op}: {name} is on {t.device}, q on {q.device}")


def _check_param(op: str, q: torch.Tensor, name: str, t: torch.Tensor) -> None:
    """A learned parameter: the dtype of q, or fp32 beside fp16 / bf16."""
    if t.device != q.device:
        raise ValueError(f"{op}: {name} is on {t.device}, q on {q.device}")
    if t.dtype != q.dtype and not (t.dtype == torch.float32
                                   and q.dtype in (torch.float16, torch.bfloat16)):
        raise TypeError(f"{op}: {name} is {t.dtype}; it has the dtype of q "
                        f"({q.dtype}), or fp32 with fp16 / bf16")


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride in its last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, acc: torch.dtype) -> torch.Tensor:
    """Cosines or sines as the kernels read them (no gradient)."""
    if t.dtype == acc and not t.requires_grad and t.is_contiguous():
        return t
    return t.detach().to(acc).contiguous()


def _tiled(t: torch.Tensor) -> torch.Tensor:
    """t in a layout the tensor-core kernels can load: unit stride in D, and for
    16-bit types a 16-byte aligned start and strides (a copy where it is not;
    the FMA kernels that read any layout would cost far more)."""
    n, s = t.shape, t.stride()
    if s[3] != 1 and n[3] != 1:
        return t.contiguous()
    if t.element_size() != 2 or n[3] % 8 or n[3] > 128:
        return t
    if t.data_ptr() % 16 == 0 and all(
            n[i] == 1 or (s[i] > 0 and s[i] % 8 == 0) for i in (0, 1, 2)):
        return t
    return t.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous from a 16-byte boundary on (what the backward of a flat
    concatenation hands out need not start on one)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _int32(op: str, name: str, t: torch.Tensor, device) -> torch.Tensor:
    if (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device
            and t.is_contiguous()):
        return t
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{op}: {name} must be an int32 or int64 tensor")
    if t.device != device:
        raise ValueError(f"{op}: {name} is on {t.device}, q on {device}")
    if t.dtype == torch.int64:   # (a wrapped position would be another one)
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(torch.int32).contiguous()


def _acc(dt: torch.dtype) -> torch.dtype:
    return torch.float64 if dt == torch.float64 else torch.float32


def _addr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# qk_norm_rotate
# ---------------------------------------------------------------------------

def _rotate_args(q, k, wq, wk, cos, sin, positions, adjacent, eps, *, with_q=True,
                 with_k=True):
    B, L, Hq, D = q.shape
    rows, half = cos.shape
    w = wq if wq is not None else wk
    code = _lib.dtype_code(q.dtype)
    return _lib.pack_norm_rotate(
        B, L, Hq * with_q, k.shape[2] * with_k, D, 2 * half, rows, *q.stride()[:3], *k.stride()[:3],
        q.data_ptr(), k.data_ptr(), _addr(wq), _addr(wk), cos.data_ptr(),
        sin.data_ptr(), _addr(positions), code,
        code if w is None else _lib.dtype_code(w.dtype), adjacent, eps)


def _rotate_fwd(q, k, wq, wk, cos, sin, positions, adjacent, eps):
    qo, ko = q.new_empty(q.shape), k.new_empty(k.shape)
    _lib.launch(q.device, "nsc_qk_norm_rotate_fwd",
                _rotate_args(q, k, wq, wk, cos, sin, positions, adjacent, eps),
                qo.data_ptr(), ko.data_ptr())
    return qo, ko


class _RotateFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, adjacent, eps):
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        ctx.adjacent, ctx.eps = adjacent, eps
        return _rotate_fwd(q, k, wq, wk, cos, sin, positions, adjacent, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        need = ctx.needs_input_grad
        dwq = torch.empty_like(wq) if wq is not None and need[2] else None
        dwk = torch.empty_like(wk) if wk is not None and need[3] else None
        # (a side that is not wanted is one of no heads)
        with_q, with_k = need[0] or dwq is not None, need[1] or dwk is not None
        dq, gq = (q.new_empty(q.shape), _aligned(gq)) if with_q else (None, None)
        dk, gk = (k.new_empty(k.shape), _aligned(gk)) if with_k else (None, None)
        a = _rotate_args(q, k, wq, wk, cos, sin, positions, ctx.adjacent, ctx.eps,
                         with_q=with_q, with_k=with_k)
        ws = None
        if dwq is not None or dwk is not None:
            ws = _lib.workspace("nsc_qk_norm_rotate_workspace", q.device, a)
        _lib.launch(q.device, "nsc_qk_norm_rotate_bwd", a, _addr(gq), _addr(gk),
                    _addr(dq), _addr(dk), _addr(dwq), _addr(dwk), _addr(ws))
        return dq, dk, dwq, dwk, None, None, None, None, None


def qk_norm_rotate(q: torch.Tensor, k: torch.Tensor,
                   q_weight: Optional[torch.Tensor],
                   k_weight: Optional[torch.Tensor], cos: torch.Tensor,
                   sin: torch.Tensor, *, positions: Optional[torch.Tensor] = None,
                   adjacent: bool = False,
                   eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """Root-mean-square norm of every head of q (B, L, Hq, D) and k
    (B, L, Hkv, D), times the weights (D,) (None: no weight), then the
    rotation by position, in one pass -> contiguous (q', k').

    cos, sin: (rows, R/2), R <= D: pair i of the first R channels -- (i,
    i + R/2), or (2i, 2i + 1) with adjacent=True -- turns by the angle of
    row positions[b, l] (int (B, L) or (L,); default: row l).  Channels past
    R are only normed.  Differentiable in q, k and the weights; the weight
    gradients are summed in a fixed order."""
    op = "qk_norm_rotate"
    _check_heads(op, "q", q)
    _check_heads(op, "k", k)
    _check_like(op, q, k=k)
    B, L, _, D = q.shape
    if k.shape[0] != B or k.shape[1] != L or k.shape[3] != D:
        raise RuntimeError(f"{op}: q {tuple(q.shape)} and k {tuple(k.shape)} "
                           f"do not agree")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        _check_param(op, q, name, w)
        if w.shape != (D,):
            raise RuntimeError(f"{op}: {name} must be ({D},); got {tuple(w.shape)}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"{op}: q_weight is {q_weight.dtype}, k_weight "
                        f"{k_weight.dtype}")
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise RuntimeError(f"{op}: cos and sin must be (rows, R/2) with R <= {D}; got "
                           f"{tuple(cos.shape)}, {tuple(sin.shape)}")
    if cos.device != q.device or sin.device != q.device:
        raise ValueError(f"{op}: cos and sin must be on {q.device}")
    _refuse_tangents(op, q, k, q_weight, k_weight, cos, sin)
    _require_cuda(op, q)
    if positions is not None:
        positions = _int32(op, "positions", positions, q.device)
        if positions.shape == (L,):
            positions = positions.expand(B, L).contiguous()
        if positions.shape != (B, L):
            raise RuntimeError(f"{op}: positions must be ({B}, {L}) or ({L},); got "
                               f"{tuple(positions.shape)}")
    elif cos.shape[0] < L:
        raise RuntimeError(f"{op}: cos and sin have {cos.shape[0]} rows for "
                           f"{L} positions")
    acc = _acc(q.dtype)
    args = (_unit(q), _unit(k), _dense(q_weight), _dense(k_weight), _table(cos, acc),
            _table(sin, acc), positions, int(adjacent), float(eps))
    if torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad
            or (q_weight is not None and q_weight.requires_grad)
            or (k_weight is not None and k_weight.requires_grad)):
        return _RotateFn.apply(*args)
    return _rotate_fwd(*args)


# ---------------------------------------------------------------------------
# token_attention
# ---------------------------------------------------------------------------

def relative_buckets(num_buckets: int, max_distance: int,
                     bidirectional: bool = True, device=None) -> torch.Tensor:
    """Bucket of every distance key - query in [-max_distance, max_distance]
    ((2 max_distance + 1,) int32; farther distances take the ends' buckets).

    Each sign has its own half of the buckets (bidirectional=False: keys past
    the query share bucket 0 and the past has all buckets).  Half of a sign's
    buckets hold one distance each, the others grow by a constant factor up to
    max_distance."""
    n = num_buckets // 2 if bidirectional else num_buckets
    if n < 2 or num_buckets > 256:
        raise ValueError(f"relative_buckets: num_buckets = {num_buckets}, need "
                         f"{4 if bidirectional else 2}..256")
    near = n // 2
    if not near < max_distance <= 1024:
        raise ValueError(f"relative_buckets: max_distance = {max_distance}, need "
                         f"{near + 1}..1024 for {num_buckets} buckets")
    rows = []
    for d in range(-max_distance, max_distance + 1):
        a = abs(d) if bidirectional else max(-d, 0)
        u = a if a < near else min(n - 1, near + int(
            math.log(a / near) / math.log(max_distance / near) * (n - near)))
        rows.append(u + (n if bidirectional and d > 0 else 0))
    return torch.tensor(rows, dtype=torch.int32, device=device)


def _attention_args(q, k, v, documents, prefix, lengths, table, buckets, scale,
                    cap, causal):
    B, Lq, Hq, D = q.shape
    code = _lib.dtype_code(q.dtype)
    docs = docs_stride = n_buckets = reach = 0
    table_code = code
    if documents is not None:
        docs, docs_stride = documents.shape[1] - 1, documents.stride(0)
    if table is not None:
        n_buckets, reach = table.shape[0], buckets.shape[0] // 2
        table_code = _lib.dtype_code(table.dtype)
    return _lib.pack_attention(
        B, Lq, k.shape[1], Hq, k.shape[2], D, *q.stride()[:3], *k.stride()[:3],
        *v.stride()[:3], docs, docs_stride, 0 if prefix is None else prefix.stride(0),
        n_buckets, reach, q.data_ptr(), k.data_ptr(), v.data_ptr(), _addr(documents),
        _addr(prefix), _addr(lengths), _addr(buckets), _addr(table), scale, cap, code,
        table_code, causal)


def _attention_fwd(q, k, v, documents, prefix, table, buckets, scale, cap, causal,
                   want_lse, train=False):
    """(out, lse or None, stats or None, residue or None)"""
    B, Lq, Hq, D = q.shape
    dev = q.device
    out = q.new_empty((B, Lq, Hq, D))
    lse = stats = residue = None
    if want_lse:
        lse = torch.empty((B, Hq, Lq), dtype=_acc(q.dtype), device=dev)
    if train:
        stats = torch.empty((2, B, Hq, Lq), dtype=_acc(q.dtype), device=dev)
        if q.element_size() == 2:
            # a score's gradient is less its row's sum of grad_out * out: with few
            # keys, or summed up in a bias bucket, what rounding out drops would show
            residue = torch.empty_like(out)
    a = _attention_args(q, k, v, documents, prefix, None, table, buckets, scale,
                        cap, causal)
    _lib.launch(dev, "nsc_token_attention_fwd", a, out.data_ptr(), _addr(lse),
                _addr(stats), _addr(residue))
    return out, lse, stats, residue


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, documents, prefix, table, buckets, scale, cap, causal,
                want_lse):
        out, lse, stats, residue = _attention_fwd(
            q, k, v, documents, prefix, table, buckets, scale, cap, causal, want_lse,
            True)
        ctx.save_for_backward(q, k, v, out, stats, residue, documents, prefix, table,
                              buckets)
        ctx.scale, ctx.cap, ctx.causal = scale, cap, causal
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_lse):
        (q, k, v, out, stats, residue, documents, prefix, table,
         buckets) = ctx.saved_tensors
        a = _attention_args(q, k, v, documents, prefix, None, table, buckets,
                            ctx.scale, ctx.cap, ctx.causal)
        grad_out = torch.zeros_like(out) if grad_out is None else _tiled(grad_out)
        if grad_lse is not None:
            grad_lse = grad_lse.contiguous()
        # the kernels give dq with the table's gradient, and dk with dv
        need = ctx.needs_input_grad
        dt = torch.empty_like(table) if table is not None and need[5] else None
        dq = q.new_empty(q.shape) if need[0] or dt is not None else None
        dk = dv = None
        if need[1] or need[2]:
            dk, dv = k.new_empty(k.shape), v.new_empty(v.shape)
        ws = _lib.workspace("nsc_token_attention_bwd_workspace", q.device, a)
        g = _lib.pack_attention_grad(
            *grad_out.stride()[:3], out.data_ptr(), stats.data_ptr(), _addr(residue),
            grad_out.data_ptr(), _addr(grad_lse), _addr(dq), _addr(dk), _addr(dv),
            _addr(dt), _addr(ws))
        _lib.launch(q.device, "nsc_token_attention_bwd", a, g)
        return dq, dk, dv, None, None, dt, None, None, None, None, None


def _check_qkv(op, q, k, v, kname="k", vname="v"):
    _check_heads(op, "q", q)
    _check_heads(op, kname, k)
    _check_heads(op, vname, v)
    _check_like(op, q, **{kname: k, vname: v})
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise RuntimeError(f"{op}: q {tuple(q.shape)}, {kname} {tuple(k.shape)} and "
                           f"{vname} {tuple(v.shape)} do not agree")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2] or q.shape[2] == 0:
        raise RuntimeError(f"{op}: {q.shape[2]} query heads are not a multiple of "
                           f"{k.shape[2]} key heads")


def _check_bias(op, q, table, buckets):
    if (table is None) != (buckets is None):
        raise ValueError(f"{op}: a bias needs bias_table and bias_buckets")
    if table is None:
        return None, None
    _check_param(op, q, "bias_table", table)
    if table.dim() != 2 or table.shape[1] != q.shape[2]:
        raise RuntimeError(f"{op}: bias_table must be (buckets, {q.shape[2]}); got "
                           f"{tuple(table.shape)}")
    buckets = _int32(op, "bias_buckets", buckets, q.device)
    if buckets.dim() != 1 or buckets.shape[0] % 2 == 0:
        raise RuntimeError(f"{op}: bias_buckets must have 2 reach + 1 entries; got "
                           f"{tuple(buckets.shape)}")
    return _dense(table), buckets


def _numbers(q, scale, softcap):
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    return scale, 0.0 if softcap is None else float(softcap)


def token_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                    scale: Optional[float] = None, softcap: Optional[float] = None,
                    causal: bool = False, prefix=None,
                    documents: Optional[torch.Tensor] = None,
                    bias_table: Optional[torch.Tensor] = None,
                    bias_buckets: Optional[torch.Tensor] = None,
                    return_lse: bool = False):
    """Softmax attention of q (B, Lq, Hq, D) over k, v (B, Lk, Hkv, D) ->
    out (B, Lq, Hq, D), or (out, lse (B, Hq, Lq) fp32).

    Query head h reads key head h Hkv // Hq; query i stands at key position
    i + Lk - Lq.  scale defaults to D^-0.5; softcap c (1e-30 to 1e30; 0 or None: none)
    turns a score s into c tanh(s / c); then bias_table[bias_buckets[distance], h] is added
    (`relative_buckets`; distances past the map's ends take the ends').

    causal: a query sees keys up to its own position.  prefix (an int, or an
    int tensor (B,), or (B, documents)): and the first `prefix` keys of its row or
    document.  documents: (B, n + 1) or (n + 1,) ascending bounds; tokens see
    only their own document, tokens outside all documents see nothing.  A query
    that sees nothing gives out = 0, lse = -inf.  What a query does not see has no
    influence on it, even where it is not finite.

    Differentiable in q, k, v and bias_table, through out and lse; the
    gradients are summed in a fixed order.  What the backward keeps beside the inputs:
    out, two numbers a row, and with fp16 / bf16 what rounding dropped of out, a second
    tensor of its size."""
    op = "token_attention"
    _check_qkv(op, q, k, v)
    B, Lq, Lk, dev = q.shape[0], q.shape[1], k.shape[1], q.device
    table, buckets = _check_bias(op, q, bias_table, bias_buckets)
    if prefix is not None and not causal:
        raise ValueError(f"{op}: a prefix needs causal=True")
    _refuse_tangents(op, q, k, v, table)
    _require_cuda(op, q)
    if documents is not None:
        documents = _int32(op, "documents", documents, dev)
        if documents.dim() == 1:
            documents = documents.expand(B, -1)
        if documents.dim() != 2 or documents.shape[0] != B or documents.shape[1] < 2:
            raise RuntimeError(f"{op}: documents must be ({B}, n + 1) or (n + 1,) bounds; "
                               f"got {tuple(documents.shape)}")
        if Lq != Lk:
            raise RuntimeError(f"{op}: documents need as many queries as keys; got "
                               f"{Lq} and {Lk}")
    if prefix is not None:
        if isinstance(prefix, int):
            prefix = torch.full((1,), prefix, dtype=torch.int32, device=dev).expand(B)
        else:
            prefix = _int32(op, "prefix", prefix, dev)
        n = 1 if documents is None else documents.shape[1] - 1
        if prefix.dim() == 1:
            prefix = prefix[:, None].expand(-1, n) if n == 1 else \
                prefix[:, None].expand(-1, n).contiguous()
        if prefix.shape != (B, n):
            raise RuntimeError(f"{op}: prefix must be ({B},) or ({B}, {n}); got "
                               f"{tuple(prefix.shape)}")
    scale, cap = _numbers(q, scale, softcap)
    train = torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or v.requires_grad
        or (table is not None and table.requires_grad))
    if (Lq <= 64 and Lk >= 256 and not train and documents is None and prefix is None
            and (causal or table is None) and _few_queries(q, k, v)):
        out, lse = _decode(q, k, v, None, table, buckets, scale, cap, int(causal),
                           return_lse)
        return (out, lse) if return_lse else out
    args = (_tiled(q), _tiled(k), _tiled(v), documents, prefix, table, buckets, scale,
            cap, int(causal), return_lse)
    if train:
        out, lse = _AttentionFn.apply(*args)
    else:
        out, lse = _attention_fwd(*args)[:2]
    return (out, lse) if return_lse else out


def _few_queries(q, k, v) -> bool:
    """Whether few queries over many keys take the decode form: its blocks hold the rows of
    all heads that share a key head, 32 at a time (fp32: 8), and share out the keys.

    Against a tile of 128 queries a head, us: 8 key heads of 64, 8192 keys, 1 / 32 queries:
    83 / 83 against 11 / 18; 8 x 8 key heads of 128, 4 queries a key, 1024 keys, 1 / 8
    queries: 22 / 23 against 12 / 27, 8192 keys: 135 / 135 against 51 / 83, 16 queries
    137 against 156; one such sequence, 64 queries, 8192 keys: 89 against 77.  fp32 (its
    tiles of FMA products), 8 such sequences, 256 keys, 16 / 32 queries: 76 / 78 against
    69 / 130; one, 1024 keys, 64 queries: 203 against 143."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    unit = 16 // q.element_size()
    if unit < 4 or D > 128 or D % unit or any(
            t.data_ptr() % 16 or t.stride(3) != 1 or any(s % unit for s in t.stride()[:3])
            for t in (q, k, v)):
        return False
    rows = Lq * (Hq // Hkv)
    if unit == 4:
        return Lq <= 16 or B * Hkv * ((rows + 7) // 8) <= 512
    return rows <= 16 or (Lk >= 2048 and (
        rows <= 32 or B * Hkv * ((rows + 31) // 32) <= 64))


def _decode(q, k, v, lengths, table, buckets, scale, cap, causal, want_lse):
    """(out, lse or None)"""
    B, T, Hq, D = q.shape
    q, k, v = _unit(q), _unit(k), _unit(v)
    out = q.new_empty((B, T, Hq, D))
    lse = (torch.empty((B, Hq, T), dtype=_acc(q.dtype), device=q.device)
           if want_lse else None)
    a = _attention_args(q, k, v, None, None, lengths, table, buckets, scale, cap, causal)
    ws = _lib.workspace("nsc_token_attention_decode_workspace", q.device, a)
    _lib.launch(q.device, "nsc_token_attention_decode", a, out.data_ptr(), _addr(lse),
                _addr(ws))
    return out, lse


def token_attention_decode(q: torch.Tensor, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, lengths: torch.Tensor, *,
                           scale: Optional[float] = None,
                           softcap: Optional[float] = None,
                           bias_table: Optional[torch.Tensor] = None,
                           bias_buckets: Optional[torch.Tensor] = None,
                           return_lse: bool = False):
    """The newest T tokens of every sequence over its cache: q (B, T, Hq, D),
    caches (B, rows, Hkv, D) whose first lengths[b] rows hold sequence b, the
    new tokens' own keys among them -> out (B, T, Hq, D) (and lse (B, Hq, T)).

    Token t stands at position lengths[b] - T + t and sees the keys up to it;
    scores as in `token_attention`.  Rows past lengths[b] are not read.  For
    serving: no gradient."""
    op = "token_attention_decode"
    _check_qkv(op, q, k_cache, v_cache, "k_cache", "v_cache")
    table, buckets = _check_bias(op, q, bias_table, bias_buckets)
    if torch.is_grad_enabled() and (
            q.requires_grad or k_cache.requires_grad or v_cache.requires_grad
            or (table is not None and table.requires_grad)):
        raise RuntimeError(f"{op} has no backward; use token_attention, or "
                           f"torch.no_grad()")
    _refuse_tangents(op, q, k_cache, v_cache, table)
    _require_cuda(op, q)
    lengths = _int32(op, "lengths", lengths, q.device)
    if lengths.shape != (q.shape[0],):
        raise RuntimeError(f"{op}: lengths must be ({q.shape[0]},); got "
                           f"{tuple(lengths.shape)}")
    scale, cap = _numbers(q, scale, softcap)
    out, lse = _decode(q, k_cache, v_cache, lengths, table, buckets, scale, cap, 1,
                       return_lse)
    return (out, lse) if return_lse else out
