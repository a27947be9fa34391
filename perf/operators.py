"""Cases of the token-attention operators, with their plain and 64-bit forms.

Three operators that a token-mixing denoiser or image language model built on
this package runs together:

  rotate     qk_norm_rotate: root-mean-square norm of every query and key head
             and the position rotation, in one pass
  attention  token_attention: softmax attention with shared key heads, scores
             capped by a tanh, a learned bias by buckets of distance, and
             causal / document / prefix masks
  decode     token_attention_decode: the same scores for the newest tokens of
             ragged sequences over a key / value cache

`run` calls the package where `own` is true, and elsewhere computes the same
results with elementary torch operations in 32 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rotate(name, dtype, B, L, Hq, Hkv, D, train=False, pairs="half", given=False):
    return {"name": name, "op": "rotate", "dtype": dtype, "B": B, "L": L, "Hq": Hq,
            "Hkv": Hkv, "D": D, "train": train, "pairs": pairs, "given": given}


def _attention(name, dtype, B, Lq, Lk, Hq, Hkv, D, train=False, cap=0.0, causal=False,
               docs=0, prefix=0, buckets=0, reach=0, layout=0):
    return {"name": name, "op": "attention", "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk,
            "Hq": Hq, "Hkv": Hkv, "D": D, "train": train, "cap": cap, "causal": causal,
            "docs": docs, "prefix": prefix, "buckets": buckets, "reach": reach,
            "layout": layout}


def _decode(name, dtype, B, T, longest, Hq, Hkv, D, cap=0.0, buckets=0, reach=0, layout=0):
    return {"name": name, "op": "decode", "dtype": dtype, "B": B, "T": T,
            "longest": longest, "Hq": Hq, "Hkv": Hkv, "D": D, "cap": cap,
            "buckets": buckets, "reach": reach, "layout": layout}


def listed():
    return [
        # one new token for each of 8 served sequences, at its own position
        _rotate("rotate_token", "bf16", 8, 1, 16, 4, 64, given=True),
        # the projections of two prompts of odd length, adjacent pairs rotated
        _rotate("rotate_prompt", "f16", 2, 2047, 32, 8, 128, pairs="adjacent"),
        # a training step over four sequences: both gradients and the norms' weights
        _rotate("rotate_train", "bf16", 4, 4096, 16, 16, 128, train=True),
        # 8 x 8 windows of 256 x 256 feature maps with a learned position bias
        _attention("windows", "f16", 256, 64, 64, 8, 8, 32, buckets=32, reach=63),
        # a long prompt through a causal layer with capped scores
        _attention("prompt_capped", "bf16", 1, 4096, 4096, 32, 8, 128, cap=20.0, causal=True),
        # images packed into one row of tokens, each with its own visible prefix
        _attention("packed_prefix", "bf16", 1, 8191, 8191, 16, 4, 64, causal=True, docs=7,
                   prefix=300, layout=3),
        # training of a layer that sees all tokens of a 64 x 32 grid, with the
        # gradient of the bias table
        _attention("train_buckets", "bf16", 4, 2048, 2048, 16, 16, 64, train=True, buckets=32,
                   reach=128),
        # training on packed documents with capped scores and shared key heads
        _attention("train_packed", "bf16", 1, 8192, 8192, 16, 4, 128, train=True, cap=30.0,
                   causal=True, docs=4, layout=5),
        # the same kind of layer in full precision, at a small odd size
        _attention("train_f32", "f32", 2, 333, 333, 4, 2, 64, train=True, causal=True,
                   buckets=16, reach=64),
        # one token for one short sequence
        _decode("decode_one", "bf16", 1, 1, 1023, 16, 4, 64),
        # one token for each of 32 ragged sequences, with capped scores
        _decode("decode_batch", "bf16", 32, 1, 8192, 32, 8, 128, cap=30.0, layout=1),
        # four drafted tokens of two long sequences, with a position bias
        _decode("decode_long", "f16", 2, 4, 65530, 16, 2, 128, buckets=32, reach=128, layout=2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    hkv = rng.choice([1, 2, 3, 4, 8])
    return hkv * rng.choice([1, 2, 4, 6, 8]), hkv


def _one(rng):
    kind = rng.choice(["rotate", "attention", "attention", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([32, 64, 64, 96, 128, 128])
    Hq, Hkv = _heads(rng)
    if kind == "rotate":
        train = rng.random() < 0.5
        L = 1 if rng.random() < 0.2 else _log(rng, 1, 8192)
        return _rotate("", dtype, _log(rng, 1, 64), L, Hq, Hkv, D, train and L > 1,
                       rng.choice(["half", "adjacent"]), rng.random() < 0.5)
    buckets, reach = (rng.choice([8, 16, 32, 64]), _log(rng, 16, 512)) if rng.random() < 0.4 \
        else (0, 0)
    cap = rng.choice([0.0, 0.0, 15.0, 30.0, 50.0])
    layout = rng.randrange(1000)
    if kind == "decode":
        return _decode("", dtype, _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 5, 8]),
                       _log(rng, 1, 65536), Hq, Hkv, D, cap, buckets, reach, layout)
    L = _log(rng, 17, 8192)
    causal = rng.random() < 0.6
    docs = _log(rng, 2, 12) if rng.random() < 0.4 else 0
    prefix = _log(rng, 1, L) if causal and rng.random() < 0.4 else 0
    train = rng.random() < 0.5
    Lq = L if train or docs or rng.random() < 0.6 else _log(rng, 1, L)
    return _attention("", dtype, _log(rng, 1, 64), Lq, L, Hq, Hkv, D, train, cap, causal, docs,
                      prefix, buckets, reach, layout)


def _fits(case):
    w = work(case)
    if case["op"] == "attention":
        scores = case["B"] * case["Hq"] * case["Lq"] * case["Lk"]
        cost = 4.0 if case["dtype"] == "f32" else 1.0
        return w["flops"] * cost <= 1.5e12 and scores <= (1 << 30) and w["bytes"] < 5e8 \
            and w["flops"] >= 1e6
    return w["bytes"] <= (5e8 if case["op"] == "rotate" else 6e8)


def draw(rng):
    while True:
        case = _one(rng)
        if _fits(case):
            case.pop("name")
            return case


# ---------------------------------------------------------------------------
# layouts: document bounds, prefixes and lengths belong to the case
# ---------------------------------------------------------------------------

def _bounds(case):
    """(B, docs + 1) document bounds; the last documents may leave padding."""
    r = random.Random("bounds %d" % case["layout"])
    rows = []
    for _ in range(case["B"]):
        end = case["Lk"] if r.random() < 0.5 else case["Lk"] - r.randrange(1 + case["Lk"] // 16)
        cuts = sorted(r.randrange(end + 1) for _ in range(case["docs"] - 1))
        rows.append([0] + cuts + [end])
    return rows


def _prefixes(case):
    """(B, docs or 1) prefix lengths, up to case["prefix"]."""
    r = random.Random("prefix %d" % case["layout"])
    return [[r.randrange(case["prefix"] // 2, case["prefix"] + 1)
             for _ in range(max(1, case["docs"]))] for _ in range(case["B"])]


def _lengths(case):
    r = random.Random("lengths %d" % case["layout"])
    out = [_log(r, max(1, case["longest"] // 8), case["longest"]) for _ in range(case["B"])]
    out[r.randrange(len(out))] = case["longest"]
    return out


def _bucket_map(n, reach):
    """Bucket of each distance key - query in [-reach, reach], both signs apart:
    half of a sign's buckets for one distance each, the others by logarithm."""
    half = n // 2
    exact_n = max(1, half // 2)
    out = []
    for d in range(-reach, reach + 1):
        a = abs(d)
        if a < exact_n:
            b = a
        else:
            top = math.log(max(2.0, reach / exact_n))
            b = min(half - 1, exact_n + int(math.log(a / exact_n) / top * (half - exact_n)))
        out.append(b + (half if d > 0 else 0))
    return out


def _spans(case):
    """Visible keys [lo, hi) of every query, as nested lists (B, Lq)."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    shift = Lk - Lq
    bounds = _bounds(case) if case["docs"] else [[0, Lk]] * B
    pre = _prefixes(case) if case["prefix"] else [[0] * max(1, case["docs"])] * B
    rows = []
    for b in range(B):
        row = [(0, 0)] * Lq
        for d in range(len(bounds[b]) - 1):
            s, e = bounds[b][d], bounds[b][d + 1]
            for p in range(max(s, shift) if case["docs"] else shift, e):
                if p - shift < 0 or p - shift >= Lq:
                    continue
                hi = min(e, max(p + 1, s + pre[b][d])) if case["causal"] else e
                row[p - shift] = (s, max(s, hi))
        rows.append(row)
    return rows


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------

def work(case):
    es = SIZES[case["dtype"]]
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    if case["op"] == "rotate":
        n = case["B"] * case["L"] * (Hq + Hkv) * D
        return {"bytes": n * es * (4 if case["train"] else 2),
                "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "decode":
        pairs = 0
        keys = 0
        for n in _lengths(case):
            keys += n
            pairs += sum(max(0, n - t) for t in range(case["T"]))
        return {"bytes": es * D * (2 * keys * Hkv + 2 * case["B"] * case["T"] * Hq),
                "flops": 4 * pairs * Hq * D}
    pairs = sum(hi - lo for row in _spans(case) for lo, hi in row)
    nq = case["B"] * case["Lq"] * Hq * D
    nk = case["B"] * case["Lk"] * Hkv * D
    # forward: q, k, v read, out written; training also reads grad_out and
    # writes grad_q, grad_k, grad_v; two products forward, four backward
    tensors = (4 * nq + 4 * nk) if case["train"] else (2 * nq + 2 * nk)
    return {"bytes": tensors * es, "flops": pairs * Hq * D * (12 if case["train"] else 4)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype, mul=1.0):
    t = torch.randn(*shape, generator=g, device="cuda")
    return t.mul_(mul).to(dtype) if mul != 1.0 else t.to(dtype)


def _projected(g, case, lq, lk, dtype, mul):
    """Queries, keys and values as a layer has them: views of one projection
    where the lengths agree."""
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    if lq == lk:
        # queries and keys at `mul`, values near one
        x = torch.randn(B, lq, Hq + 2 * Hkv, D, generator=g, device="cuda")
        x[:, :, :Hq + Hkv] *= mul
        x = x.to(dtype)
        return x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
    return (_randn(g, B, lq, Hq, D, dtype=dtype, mul=mul),
            _randn(g, B, lk, Hkv, D, dtype=dtype, mul=mul),
            _randn(g, B, lk, Hkv, D, dtype=dtype))


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    st = {"case": case}
    if case["op"] == "rotate":
        L = case["L"]
        st["q"], st["k"], _ = _projected(g, case, L, L, dt, 1.7)
        st["q_weight"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
        st["k_weight"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
        rows = max(L, 16384 if case["given"] else L)
        freq = 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["positions"] = (torch.randint(0, rows - L + 1, (B, 1), generator=g, device="cuda")
                           + torch.arange(L, device="cuda")).to(torch.int32) \
            if case["given"] else None
        if case["train"]:
            st["grad_q"] = _randn(g, B, L, Hq, D, dtype=dt)
            st["grad_k"] = _randn(g, B, L, Hkv, D, dtype=dt)
        return st
    if case["buckets"]:
        st["table"] = _randn(g, case["buckets"], Hq, dtype=dt)
        st["map"] = torch.tensor(_bucket_map(case["buckets"], case["reach"]), dtype=torch.int32,
                                 device="cuda")
    else:
        st["table"] = st["map"] = None
    st["scale"] = D ** -0.5
    if case["op"] == "decode":
        n = case["longest"]
        st["q"] = _randn(g, B, case["T"], Hq, D, dtype=dt, mul=1.3)
        st["k"] = _randn(g, B, n, Hkv, D, dtype=dt, mul=1.3)
        st["v"] = _randn(g, B, n, Hkv, D, dtype=dt)
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        return st
    st["q"], st["k"], st["v"] = _projected(g, case, case["Lq"], case["Lk"], dt, 1.5)
    st["documents"] = torch.tensor(_bounds(case), dtype=torch.int32, device="cuda") \
        if case["docs"] else None
    st["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda") \
        if case["prefix"] else None
    if case["train"]:
        st["grad_out"] = _randn(g, B, case["Lq"], Hq, D, dtype=dt)
    return st


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_rotate_one(x, weight, cos, sin, adjacent):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    if adjacent:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_rotate(q, k, wq, wk, st):
    case = st["case"]
    L = case["L"]
    if st["positions"] is None:
        cos, sin = st["cos"][:L, None], st["sin"][:L, None]
    else:
        at = st["positions"].long()
        cos, sin = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
    adjacent = case["pairs"] == "adjacent"
    return (_plain_rotate_one(q, wq, cos, sin, adjacent).to(q.dtype),
            _plain_rotate_one(k, wk, cos, sin, adjacent).to(k.dtype))


def _plain_mask(st, Lq, Lk):
    """(B or 1, 1, 1, Lq, Lk) visible pairs, or None where all are."""
    case = st["case"]
    dev = st["q"].device
    key = torch.arange(Lk, device=dev)
    query = torch.arange(Lq, device=dev) + (Lk - Lq)
    seen = None
    start = torch.zeros(1, 1, dtype=torch.long, device=dev)
    pre = st["prefix"]
    if st["documents"] is not None:
        doc = st["documents"].long()
        at = (key[None, :, None] >= doc[:, None, :]).sum(-1) - 1            # (B, L)
        inside = (at >= 0) & (at < doc.shape[1] - 1)
        one = at.clamp(0, doc.shape[1] - 2)
        seen = (one[:, :, None] == one[:, None, :]) & inside[:, :, None] & inside[:, None, :]
        start = doc.gather(1, one)
        if pre is not None:
            pre = pre.long().gather(1, one)
    if case["causal"]:
        ok = (key[None, :] <= query[:, None])[None]
        if pre is not None:
            ok = ok | (key[None, None, :] < (start + pre)[:, :, None])
        seen = ok if seen is None else seen & ok
    return None if seen is None else seen[:, None, None]


def _plain_bias(st, Lq, Lk):
    """(1, Hkv, G, Lq, Lk) bias: a vector over distances, laid out along the
    diagonals by reshapes alone (its gradient is then a sum, in one order)."""
    case = st["case"]
    n = Lq + Lk - 1
    rel = torch.arange(n, device=st["q"].device)
    rel = torch.where(rel < Lk, rel, rel - n) - (Lk - Lq)
    one = st["map"].long()[rel.clamp(-case["reach"], case["reach"]) + case["reach"]]
    pick = (one[:, None] == torch.arange(case["buckets"], device=rel.device)).float()
    vec = st["table"].float().t() @ pick.t()                                # (Hq, n)
    H = vec.shape[0]
    if n == 1:
        full = vec[:, None]
    else:
        full = vec[:, None].expand(H, Lq, n).reshape(H, Lq * n)[:, :Lq * (n - 1)]
        full = full.reshape(H, Lq, n - 1)
        full = full[:, :, :Lk] if n - 1 >= Lk else torch.cat([full, vec[:, None, n - 1:]], -1)
    return full.reshape(1, case["Hkv"], H // case["Hkv"], Lq, Lk)


def _plain_scores(q, k, st):
    case = st["case"]
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    qf = q.float().transpose(1, 2).reshape(B, Hkv, Hq // Hkv * Lq, D)
    s = (qf @ k.float().permute(0, 2, 3, 1)).reshape(B, Hkv, Hq // Hkv, Lq, Lk) * st["scale"]
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    return s


def _plain_mix(s, seen, v, dtype):
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    B, Hkv, G, Lq, Lk = p.shape
    o = p.reshape(B, Hkv, G * Lq, Lk) @ v.float().transpose(1, 2)
    o = o.reshape(B, Hkv, G, Lq, -1) / torch.where(total > 0, total, torch.ones_like(total))
    return o.flatten(1, 2).transpose(1, 2).to(dtype)


def _plain_attention(q, k, v, st):
    Lq, Lk = q.shape[1], k.shape[1]
    s = _plain_scores(q, k, st)
    if st["table"] is not None:
        s = s + _plain_bias(st, Lq, Lk)
    return _plain_mix(s, _plain_mask(st, Lq, Lk), v, q.dtype)


def _plain_decode(st):
    case = st["case"]
    q, k, v = st["q"], st["k"], st["v"]
    T, n, Hkv = case["T"], case["longest"], case["Hkv"]
    s = _plain_scores(q, k, st)
    at = st["lengths"].long()[:, None] - T + torch.arange(T, device=q.device)     # (B, T)
    rel = torch.arange(n, device=q.device) - at[:, :, None]                       # (B, T, n)
    if st["table"] is not None:
        one = st["map"].long()[rel.clamp(-case["reach"], case["reach"]) + case["reach"]]
        bias = st["table"].float()[one].permute(0, 3, 1, 2)                       # (B, Hq, T, n)
        s = s + bias.reshape(bias.shape[0], Hkv, -1, T, n)
    return _plain_mix(s, (rel <= 0)[:, None, None], v, q.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own_rotate(q, k, wq, wk, st):
    import neural_shift_cuda_b200 as nsc
    return nsc.qk_norm_rotate(q, k, wq, wk, st["cos"], st["sin"], positions=st["positions"],
                              adjacent=st["case"]["pairs"] == "adjacent", eps=EPS)


def _own_attention(q, k, v, st):
    import neural_shift_cuda_b200 as nsc
    return nsc.token_attention(q, k, v, scale=st["scale"], softcap=st["case"]["cap"],
                               causal=st["case"]["causal"], documents=st["documents"],
                               prefix=st["prefix"], bias_table=st["table"],
                               bias_buckets=st["map"])


def _own_decode(st):
    import neural_shift_cuda_b200 as nsc
    return nsc.token_attention_decode(st["q"], st["k"], st["v"], st["lengths"],
                                      scale=st["scale"], softcap=st["case"]["cap"],
                                      bias_table=st["table"], bias_buckets=st["map"])


def run(state):
    case = state["case"]
    if case["op"] == "decode":
        with torch.no_grad():
            return {"out": _own_decode(state) if own else _plain_decode(state)}
    if case["op"] == "rotate":
        f = _own_rotate if own else _plain_rotate
        args = [state["q"], state["k"], state["q_weight"], state["k_weight"]]
        if not case["train"]:
            with torch.no_grad():
                q, k = f(*args, state)
            return {"q": q, "k": k}
        args = [t.detach().requires_grad_() for t in args]
        q, k = f(*args, state)
        grads = torch.autograd.grad([q, k], args, [state["grad_q"], state["grad_k"]])
        return {"q": q.detach(), "k": k.detach(), "grad_q": grads[0], "grad_k": grads[1],
                "grad_q_weight": grads[2], "grad_k_weight": grads[3]}
    f = _own_attention if own else _plain_attention
    if not case["train"]:
        with torch.no_grad():
            return {"out": f(state["q"], state["k"], state["v"], state)}
    args = [state[n].detach().requires_grad_() for n in ("q", "k", "v")]
    st = dict(state)
    if state["table"] is not None:
        st["table"] = state["table"].detach().requires_grad_()
        args.append(st["table"])
    out = f(*args[:3], st)
    grads = torch.autograd.grad(out, args, state["grad_out"])
    got = {"out": out.detach(), "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}
    if state["table"] is not None:
        got["grad_table"] = grads[3]
    return got


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_rotate(case, st):
    """The rotation as a product of complex numbers; gradients by formula."""
    B, L, D = case["B"], case["L"], case["D"]
    at = st["positions"].long() if st["positions"] is not None \
        else torch.arange(L, device="cuda").expand(B, L)
    turn = torch.complex(st["cos"].double()[at], st["sin"].double()[at])[:, :, None]
    half = D // 2

    def pair(t):
        if case["pairs"] == "adjacent":
            return torch.complex(t[..., 0::2].contiguous(), t[..., 1::2].contiguous())
        return torch.complex(t[..., :half].contiguous(), t[..., half:].contiguous())

    def unpair(z):
        if case["pairs"] == "adjacent":
            return torch.view_as_real(z).flatten(-2)
        return torch.cat([z.real, z.imag], -1)

    got = {}
    for n in ("q", "k"):
        x, w = st[n].double(), st[n + "_weight"].double()
        r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
        got[n] = unpair(pair(x * r * w) * turn)
        if case["train"]:
            h = unpair(pair(st["grad_" + n].double()) * turn.conj())
            got["grad_%s_weight" % n] = (h * x * r).sum((0, 1, 2))
            hw = h * w
            got["grad_" + n] = r * hw - x * r ** 3 * (hw * x).sum(-1, keepdim=True) / D
    return got


def _exact_bias(case, st, h, rel):
    reach = case["reach"]
    one = st["map"].long()[rel.clamp(-reach, reach) + reach]
    return st["table"].double()[:, h][one], one


def _exact_attention(case, st):
    B, Lq, Lk, Hq, Hkv = case["B"], case["Lq"], case["Lk"], case["Hq"], case["Hkv"]
    D, cap = case["D"], case["cap"]
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64, device="cuda")
    if case["train"]:
        dq = torch.zeros_like(out)
        dk = torch.zeros(B, Lk, Hkv, D, dtype=torch.float64, device="cuda")
        dv = torch.zeros_like(dk)
        dt = torch.zeros(max(1, case["buckets"]), Hq, dtype=torch.float64, device="cuda")
    spans = torch.tensor(_spans(case), device="cuda")                     # (B, Lq, 2)
    key = torch.arange(Lk, device="cuda")
    rel = key[None, :] - (torch.arange(Lq, device="cuda")[:, None] + (Lk - Lq))
    step = max(1, min(B, (1 << 26) // (Lq * Lk)))
    for b in range(0, B, step):
        e = min(B, b + step)
        hidden = (key < spans[b:e, :, :1]) | (key >= spans[b:e, :, 1:])
        for h in range(Hq):
            q = st["q"][b:e, :, h].double()
            k = st["k"][b:e, :, h * Hkv // Hq].double()
            v = st["v"][b:e, :, h * Hkv // Hq].double()
            s = torch.einsum("bqd,bkd->bqk", q, k) * st["scale"]
            if cap:
                t = torch.tanh(s / cap)
                s = t * cap
            if case["buckets"]:
                bias, one = _exact_bias(case, st, h, rel)
                s = s + bias
            s[hidden] = -math.inf
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            del s
            out[b:e, :, h] = torch.einsum("bqk,bkd->bqd", p, v)
            if not case["train"]:
                continue
            g = st["grad_out"][b:e, :, h].double()
            dv[b:e, :, h * Hkv // Hq] += torch.einsum("bqk,bqd->bkd", p, g)
            dp = torch.einsum("bqd,bkd->bqk", g, v)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            if case["buckets"]:
                flat = ds.sum(0)
                for i in range(case["buckets"]):
                    dt[i, h] += flat[one == i].sum()
            if cap:
                ds = ds * (1 - t * t)
            ds = ds * st["scale"]
            dq[b:e, :, h] = torch.einsum("bqk,bkd->bqd", ds, k)
            dk[b:e, :, h * Hkv // Hq] += torch.einsum("bqk,bqd->bkd", ds, q)
    if not case["train"]:
        return {"out": out}
    got = {"out": out, "grad_q": dq, "grad_k": dk, "grad_v": dv}
    if case["buckets"]:
        got["grad_table"] = dt
    return got


def _exact_decode(case, st):
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    out = torch.zeros(B, T, Hq, case["D"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        rel = torch.arange(n, device="cuda")[None, :] \
            - (n - T + torch.arange(T, device="cuda"))[:, None]
        for h in range(Hq):
            k = st["k"][b, :n, h * Hkv // Hq].double()
            v = st["v"][b, :n, h * Hkv // Hq].double()
            s = st["q"][b, :, h].double() @ k.t() * st["scale"]
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if case["buckets"]:
                s = s + _exact_bias(case, st, h, rel)[0]
            s[rel > 0] = -math.inf
            out[b, :, h] = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v
    return {"out": out}


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rotate": _exact_rotate, "attention": _exact_attention,
                "decode": _exact_decode}[case["op"]](case, st)
