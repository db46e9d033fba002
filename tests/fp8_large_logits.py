"""Inputs with one winning key per row and logits of chosen size, made on the CPU, and their results in 64 bits."""

from __future__ import annotations

import torch

import fp8_model as F

E4M3 = torch.float8_e4m3fn
HEADS = [(14, 2, 64), (32, 8, 128), (16, 1, 128), (24, 2, 64)]
# dtype, softmax scale, size of the query's elements and of the keys', sign of the logits.  With D products of 1 to 2
# times the two sizes each, logits in powers of two are D * 1.44 * scale * sizes and more: 2^24 to 2^40.
CASES = {
    "2^24": (torch.bfloat16, 2.0 ** 17, 1.0, 1.0, 1),
    "2^28": (torch.float16, 2.0 ** 21, 1.0, 1.0, 1),
    "2^31": (torch.bfloat16, 2.0 ** 24, 1.0, 1.0, 1),
    "2^40": (torch.float16, 2.0 ** 33, 1.0, 1.0, 1),
    "negative": (torch.bfloat16, 2.0 ** 22, 1.0, 1.0, -1),
    "negative 2^40": (torch.float16, 2.0 ** 33, 1.0, 1.0, -1),
    "negative scale": (torch.bfloat16, -2.0 ** 25, 1.0, 1.0, 1),
    "f16 rows": (torch.float16, 0.125, 12000.0, 6000.0, 1),
    "bf16 rows": (torch.bfloat16, 0.125, 3e6, 3000.0, 1),
}


def case(name, spans, heads, bs, seed=0):
    """spans: (length, rows) of each sequence.  Keys lie along one direction per KV head, `r` times as long: up to 1.5
    and one of 2 in each 200 or so (for negative logits: from 1.3 on, and one of 1)."""
    dtype, scale, qsize, ksize, sign = CASES[name]
    H, KH, D = heads
    g = torch.Generator().manual_seed(seed + sum(map(ord, name)))
    need = [-(-n // bs) for n, _ in spans]
    num_blocks = sum(need) + 3
    perm = torch.randperm(num_blocks, generator=g)
    table = torch.full((len(spans), max(need)), -1, dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    u = torch.sign(torch.randn(KH, D, generator=g)) * (1 + torch.rand(KH, D, generator=g))
    k = torch.zeros(num_blocks, KH, bs, D)
    low = sign * scale < 0
    for i, (n, _) in enumerate(spans):
        r = (1.3 + 0.7 * torch.rand(n, generator=g)) if low else 1.5 * torch.rand(n, generator=g)
        r[torch.randint(0, n, (1 + n // 200,), generator=g)[:1]] = 1.0 if low else 2.0
        pos = torch.arange(n)
        k[table[i][pos // bs], :, pos % bs] = sign * r[:, None, None] * u
    k *= 1 + 0.02 * torch.randn(k.shape, generator=g)
    k *= ksize
    v = torch.randn(num_blocks, KH, bs, D, generator=g) * torch.exp2(
        torch.randint(-5, 6, (num_blocks, KH, 1, 1), generator=g).float())
    caches, scales = [], []
    for x in (k, v):
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)).clamp_min(2.0 ** -80) / 448.0)))
        caches.append((x / s[..., None, None]).to(E4M3))
        scales.append(s)
    rows = sum(n for _, n in spans)
    q = u.repeat_interleave(H // KH, 0) * (1 + 0.05 * torch.randn(rows, H, D, generator=g)) * qsize
    return q.to(dtype), caches[0], caches[1], torch.stack(scales, -1).contiguous(), table, scale


def winners(q, kc, vc, sc, blocks, length, bs, scale):
    """For the last len(q) positions of a sequence: the value of each row's largest logit, [R, H, D]; whether it is
    larger than any other by what decides, [R, H]; and the largest value.

    A float32 logit in powers of two is off by E <= (D + 4) 2^-23 sum |q k| and a few 2^-24 of itself where it is
    scaled and subtracted, which are less; a key that is 4 E + 64 below weighs less than 2^-60."""
    R, H, D = q.shape
    blocks = blocks[:-(-length // bs)]
    k, v = (F.dequant(c, sc, w, blocks, length).repeat_interleave(H // c.shape[1], 0) for w, c in enumerate((kc, vc)))
    qd = q.double().transpose(0, 1)
    c = abs(scale) * 1.4426950408889634
    x = torch.matmul(qd, k.transpose(1, 2)) * scale * 1.4426950408889634
    E = c * (D + 4) * 2.0 ** -23 * torch.matmul(qd.abs(), k.abs().transpose(1, 2))
    seen = torch.arange(length) < (length - R + 1 + torch.arange(R))[:, None]
    x = x.masked_fill(~seen, -torch.inf)
    E = E.masked_fill(~seen, 0.0).amax(-1)
    top, at = x.max(-1)
    second = x.scatter(-1, at[..., None], -torch.inf).amax(-1)
    ref = v.gather(1, at[..., None].expand(-1, -1, D))
    return ref.transpose(0, 1), (top - second > 4 * E + 64).T, v.abs().max()
