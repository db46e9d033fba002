"""The 8-bit cache's operators in 64 bits, on the device of their inputs (a plain model for the tests)."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def scale_for(amax: float) -> float:
    """The smallest power of two s >= 2**-100 with amax <= 448 s."""
    if amax == 0:
        return 2.0 ** -100
    e = math.ceil(math.log2(amax / 448.0))
    while 448.0 * 2.0 ** e < amax:
        e += 1
    while e > -100 and 448.0 * 2.0 ** (e - 1) >= amax:
        e -= 1
    return 2.0 ** max(e, -100)


def to_codes(x: torch.Tensor) -> torch.Tensor:
    """Bytes of the nearest e4m3 values, ties to even, saturating; NaN to 0x7f.  Found by search among all values."""
    codes = torch.arange(127, dtype=torch.uint8, device=x.device)  # 0 .. 448
    grid = codes.view(E4M3).double()
    a = x.abs().double().clamp_max(448.0)
    hi = torch.searchsorted(grid, a.contiguous()).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    dl, dh = a - grid[lo], grid[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).to(torch.uint8)
    pick |= torch.signbit(x).to(torch.uint8) << 7
    return torch.where(torch.isnan(x), 0x7F, pick)


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """The rotation rounded once to float32: [T, heads, D]."""
    x = x.double()
    half = x.shape[-1] // 2
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return (x * c + turned * s).float()


def write(key, value, key_cache, value_cache, kv_scale, slots, block_size) -> None:
    """Block by block; key / value float32 [T, KH, D], caches and scales updated in place."""
    slots = slots.tolist()
    blocks = {}
    for t, s in enumerate(slots):
        if s >= 0:
            blocks.setdefault(s // block_size, {})[s % block_size] = t
    for b, rows in blocks.items():
        off = torch.tensor(sorted(rows), device=key.device)
        tok = torch.tensor([rows[o] for o in sorted(rows)], device=key.device)
        others = torch.tensor([o for o in range(block_size) if o not in rows], dtype=torch.long, device=key.device)
        for which, (x, cache) in enumerate(((key, key_cache), (value, value_cache))):
            codes = cache.view(torch.uint8)
            for h in range(x.shape[1]):
                new = x[tok, h].double()
                old = float(kv_scale[b, h, which])
                base = old if 0 not in rows and math.isfinite(old) and old > 0 else 0.0
                finite = new[torch.isfinite(new)]
                s = max(base, scale_for(float(finite.abs().max()) if finite.numel() else 0.0))
                if base > 0 and s > base and others.numel():
                    codes[b, h, others] = to_codes(codes[b, h, others].view(E4M3).double() * (base / s))
                codes[b, h, off] = to_codes(new / s)
                kv_scale[b, h, which] = s


def dequant(cache, kv_scale, which, blocks, length) -> torch.Tensor:
    """[KH, length, D] float64 of one sequence's blocks."""
    x = cache.view(torch.uint8)[blocks].view(E4M3).double() * kv_scale[blocks, :, which].double()[..., None, None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :length]


def attend(q, k, v, first, scale):
    """Rows q [R, H, D], row r attending positions < first + r: (out, tolerance), both [R, H, D].

    The tolerance counts, with A = sum p |v| / sum p and N positions:
      * p rounded to f16: 2^-11 A, and 2^-25 max|v| each for those below f16's normal range (sum p >= 1);
      * a logit in powers of two is D float32 products added up, scaled twice: off by E <= (D + 4) 2^-23
        sum |q k|, which changes numerator and denominator: 2 E A; the same for the query's elements below
        2^-14 of the row's largest (2^-25 of it each);
      * exp2, float32 sums over N positions: (N + 16) 2^-23 A.
    The output's own rounding is added by `check`.
    """
    R, H, D = q.shape
    group = H // k.shape[0]
    q = q.double().transpose(0, 1)  # [H, R, D]
    k, v = (x.repeat_interleave(group, 0) for x in (k, v))
    N = k.shape[1]
    x = torch.matmul(q, k.transpose(1, 2)) * scale
    seen = torch.arange(N, device=q.device) < (first + torch.arange(R, device=q.device))[:, None]
    x = x.masked_fill(~seen, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total
    A = torch.matmul(p, v.abs()) / total
    prod = torch.matmul(q.abs(), k.abs().transpose(1, 2)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    lost = (q.abs().amax(-1, keepdim=True) * 2.0 ** -25) * k.abs().sum(-1).amax(-1)[:, None, None]
    E = abs(scale) * ((D + 4) * 2.0 ** -23 * prod + lost)
    tol = (2.0 ** -11 + 2 * E + (N + 16) * 2.0 ** -23) * A + N * 2.0 ** -25 * v.abs().amax((1, 2))[:, None, None]
    return out.transpose(0, 1), tol.transpose(0, 1)


def check(got, ref, tol) -> None:
    assert torch.isfinite(got).all()
    d = (got.double() - ref).abs()
    limit = tol + UNIT[got.dtype] * (ref.abs() + tol) + 2.0 ** -25  # (f16's smallest step)
    worst = (d / limit).max().item()
    assert worst <= 1.0, f"{worst:.3f} of the tolerance (largest difference {d.max().item():.3e})"
