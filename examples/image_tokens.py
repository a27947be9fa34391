"""Denoising images token by token: the token operators in one small model.

Images are cut into patches, a patch is a token.  A document is one image: its
noisy patches, which see one another (the prefix), then its clean patches; the noise
of each patch is predicted from all before it.  Training packs several documents into one row;
serving denoises a batch of images with a cache, one new patch a step.

    qk_norm_rotate          norm and rotation of queries and keys, read in place
                            from one projection
    token_attention         training (packed documents, prefixes, capped scores,
                            a learned bias by distance) and the prompt
    token_attention_decode  the same scores for the newest patch over the cache

    python examples/image_tokens.py [--steps 400] [--images 8] [--dtype bf16]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import neural_shift_cuda_b200 as nsc  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Cache:
    """Keys (rotated) and values of the tokens so far, (B, rows, Hkv, D)."""

    def __init__(self, B, rows, heads, width, device, dtype):
        self.k = torch.zeros(B, rows, heads, width, device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)

    def write(self, at, k, v):
        """Tokens k, v (B, L, Hkv, D) at rows at (B, L)."""
        b = torch.arange(k.shape[0], device=k.device)[:, None]
        self.k[b, at] = k
        self.v[b, at] = v


class TokenMixer(nn.Module):
    """Attention over tokens, with a residual: queries of `heads`, keys and
    values of `key_heads` heads, all of `width` channels."""

    def __init__(self, dim, heads, key_heads, width, rows, softcap=30.0, buckets=32,
                 reach=128):
        super().__init__()
        self.shape = (heads, key_heads, width)
        self.softcap = softcap
        self.norm = nn.LayerNorm(dim)
        self.qkv = nn.Linear(dim, (heads + 2 * key_heads) * width, bias=False)
        self.out = nn.Linear(heads * width, dim, bias=False)
        self.q_weight = nn.Parameter(torch.ones(width))
        self.k_weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(buckets, heads))
        angles = torch.arange(rows)[:, None] * 1e4 ** (-torch.arange(0, width, 2) / width)
        self.register_buffer("cos", angles.cos(), persistent=False)
        self.register_buffer("sin", angles.sin(), persistent=False)
        self.register_buffer("buckets", nsc.relative_buckets(buckets, reach),
                             persistent=False)

    def _apply(self, fn, *args, **kwargs):
        # the rotation's tables stay in 32 bits where parameters are rounded: an
        # angle's error grows with the position
        tables = self.cos, self.sin
        super()._apply(fn, *args, **kwargs)
        self.cos, self.sin = (t.to(self.buckets.device) for t in tables)
        return self

    def forward(self, x, positions, *, documents=None, prefix=None, cache=None,
                lengths=None):
        """x (B, L, dim), positions (B, L) inside each document.  With a cache the
        tokens' keys and values are written to it; with lengths too, the tokens are
        the newest of each sequence and see its cache."""
        h, hk, d = self.shape
        y = self.qkv(self.norm(x).to(x.dtype)).unflatten(-1, (h + 2 * hk, d))
        q, k, v = y.split((h, hk, hk), dim=2)
        q, k = nsc.qk_norm_rotate(q, k, self.q_weight, self.k_weight, self.cos, self.sin,
                                  positions=positions)
        if cache is not None:
            cache.write(positions, k, v)
        scores = dict(softcap=self.softcap, bias_table=self.bias,
                      bias_buckets=self.buckets)
        if lengths is None:
            o = nsc.token_attention(q, k, v, causal=True, prefix=prefix,
                                    documents=documents, **scores)
        else:
            o = nsc.token_attention_decode(q, cache.k, cache.v, lengths, **scores)
        return x + self.out(o.flatten(2))


class ImageTokens(nn.Module):
    """Layers of TokenMixer and a pointwise network over patches of `patch` values."""

    def __init__(self, patch, dim=256, heads=8, key_heads=2, width=32, layers=2, rows=1024):
        super().__init__()
        self.enter = nn.Linear(patch + 1, dim)
        self.mix = nn.ModuleList(TokenMixer(dim, heads, key_heads, width, rows)
                                 for _ in range(layers))
        self.point = nn.ModuleList(
            nn.Sequential(nn.LayerNorm(dim), nn.Linear(dim, 4 * dim), nn.GELU(),
                          nn.Linear(4 * dim, dim)) for _ in range(layers))
        self.leave = nn.Linear(dim, patch)

    def forward(self, tokens, positions, *, caches=None, **where):
        x = self.enter(tokens)
        for i, (mix, point) in enumerate(zip(self.mix, self.point)):
            x = mix(x, positions, cache=caches[i] if caches else None, **where)
            x = x + point(x)
        return self.leave(x)

    def caches(self, B, rows):
        w = self.enter.weight
        return [Cache(B, rows, m.shape[1], m.shape[2], w.device, w.dtype)
                for m in self.mix]


def patches(images, size):
    """(B, H, W) -> (B, tokens, size * size)"""
    return F.unfold(images[:, None], size, stride=size).transpose(1, 2)


def shapes(n, side, generator, device):
    """n images of smooth waves, and the same with noise."""
    at = torch.linspace(0, 1, side, device=device)
    f = 6 * torch.rand(n, 2, 1, 1, generator=generator, device=device)
    clean = torch.sin(f[:, 0] * at[:, None] * 3 + f[:, 1] * at * 3)
    return clean, clean + 0.5 * torch.randn(clean.shape, generator=generator,
                                            device=device)


def marked(x, clean):
    """Tokens with a channel that tells clean patches from noisy ones."""
    return torch.cat([x, torch.full_like(x[..., :1], float(clean))], -1)


def packed(pairs, dtype):
    """Images of differing sizes as one row of documents: tokens (1, L, p + 1),
    positions, documents, prefixes, and which tokens predict what correction."""
    tokens, positions, bounds, prefix, target, predicts = [], [], [0], [], [], []
    for clean, noisy in pairs:                              # (n, p) each
        n = noisy.shape[0]
        tokens += [marked(noisy, False), marked(clean[:-1], True)]
        length = 2 * n - 1
        positions.append(torch.arange(length))
        bounds.append(bounds[-1] + length)
        prefix.append(n)
        # the last noisy patch predicts for the first clean one, and so on
        predicts.append(torch.arange(length) >= n - 1)
        target.append(clean - noisy)
    dev = tokens[0].device

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)[None]
    return (torch.cat(tokens)[None].to(dtype), torch.cat(positions)[None].to(dev),
            ints(bounds), ints(prefix), torch.cat(predicts).to(dev), torch.cat(target))


def train(model, steps, dtype, images, generator, size=4, lr=1e-3):
    """Losses of `steps` steps, each on `images` images of differing sizes."""
    dev = model.enter.weight.device
    master = [p.detach().float().clone().requires_grad_() for p in model.parameters()]
    opt = torch.optim.AdamW(master, lr=lr)
    losses = []
    for step in range(steps):
        pairs = []
        for i in range(images):
            clean, noisy = shapes(1, size * (6 + (step + i) % 3), generator, dev)
            pairs.append((patches(clean, size)[0], patches(noisy, size)[0]))
        tokens, positions, documents, prefix, predicts, target = packed(pairs, dtype)
        out = model(tokens, positions, documents=documents, prefix=prefix)
        loss = F.mse_loss(out[0, predicts].float(), target)
        model.zero_grad(set_to_none=True)
        loss.backward()
        for m, p in zip(master, model.parameters()):
            m.grad = p.grad.float()
        opt.step()
        with torch.no_grad():
            for m, p in zip(master, model.parameters()):
                p.copy_(m)
        losses.append(loss.item())
    return losses


@torch.no_grad()
def denoise(model, noisy):
    """noisy (B, n, p) patches -> clean (B, n, p): the prompt in one call, then a
    patch a step over the cache."""
    B, n, _ = noisy.shape
    dev, dtype = noisy.device, model.enter.weight.dtype
    caches = model.caches(B, 2 * n)
    at = torch.arange(n, device=dev).expand(B, n)
    x = model(marked(noisy, False).to(dtype), at, prefix=n, caches=caches)[:, -1:]
    x = x + noisy[:, :1]
    done = [x]
    lengths = torch.full((B,), n, dtype=torch.int32, device=dev)
    for i in range(n, 2 * n - 1):
        lengths += 1
        at = torch.full((B, 1), i, device=dev)
        x = model(marked(x, True).to(dtype), at, caches=caches, lengths=lengths)
        x = x + noisy[:, i - n + 1:i - n + 2]
        done.append(x)
    return torch.cat(done, 1)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--images", type=int, default=8, help="documents a row")
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    args = ap.parse_args(argv)
    if not torch.cuda.is_available():
        raise SystemExit("image_tokens: needs a CUDA device")
    dev, dtype, size = torch.device("cuda:0"), DTYPES[args.dtype], 4
    torch.manual_seed(0)
    g = torch.Generator(device=dev).manual_seed(0)
    model = ImageTokens(size * size).to(dev, dtype)
    losses = train(model, args.steps, dtype, args.images, g, size)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {args.steps} steps")
    clean, noisy = shapes(16, 28, g, dev)
    out = denoise(model, patches(noisy, size))
    target = patches(clean, size)
    print(f"mean squared error: noisy {F.mse_loss(patches(noisy, size), target):.4f}, "
          f"denoised {F.mse_loss(out.float(), target):.4f}")


if __name__ == "__main__":
    main()
