"""Attention over the 8-bit cache where logits are finite and very large: it ends, and the largest key's value comes
out (tests/test_fp8_large_logits_cpu.py has the arithmetic)."""

from __future__ import annotations

import math

import pytest
import torch

import fp8_model as F
import mini_vllm_b200 as M
from fp8_large_logits import CASES, HEADS, case, winners

DEV = torch.device("cuda", 0)


def check(out, q, kc, vc, sc, table, spans, bs, scale):
    """Rows with a winner hold its value: off by P's rounding to f16 (2^-11), which numerator and denominator do not
    share, float32 sums (2^-20 is ample) and the output's own.  The others lie between the values."""
    at = 0
    for i, (length, rows) in enumerate(spans):
        ref, sure, most = winners(q[at:at + rows], kc, vc, sc, table[i], length, bs, scale)
        got = out[at:at + rows].double().cpu()
        assert torch.isfinite(got).all()
        unit = F.UNIT[out.dtype]
        off = (2.0 ** -11 + 2.0 ** -20) * ref.abs()
        limit = torch.where(sure[..., None], off + unit * (ref.abs() + off) + 2.0 ** -25, math.inf)
        assert ((got - ref).abs() <= limit).all()
        assert (got.abs() <= most * (1 + 2.0 ** -7) + 2.0 ** -25).all()
        at += rows


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("name", list(CASES))
def test_decode(name, heads):
    lens = [700, 1, 40, 17, 333]
    q, kc, vc, sc, table, scale = case(name, [(n, 1) for n in lens], heads, 16)
    kvl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    dev = [x.to(DEV) for x in (q, kc, vc, sc, table)]
    wide = torch.cat([dev[4], torch.full((5, 400), -1, dtype=torch.int64, device=DEV)], 1)
    # units cut between CTAs (as a wide table may need), and (a narrow table, short sequences) whole ones
    for keep in (slice(0, 5), slice(1, 4)):
        sub = wide if keep.start == 0 else dev[4][keep, :3].contiguous()
        out = M.paged_decode_attention_fp8(dev[0][keep], *dev[1:4], sub, kvl[keep], 16, scale=scale)
        check(out, q[keep], kc, vc, sc, table[keep], [(n, 1) for n in lens[keep]], 16, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
def test_decode_logits_that_overflow(heads):
    """Logits below float32's range count for nothing; other sequences of the batch are as ever."""
    lens = [300, 45]
    q, kc, vc, sc, table, _ = case("negative", [(n, 1) for n in lens], heads, 16)
    scale = 2e37
    q[1] *= 1e-33
    kvl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = M.paged_decode_attention_fp8(*(x.to(DEV) for x in (q, kc, vc, sc, table)), kvl, 16, scale=scale)
    assert (out[0] == 0).all()
    check(out[1:], q[1:], kc, vc, sc, table[1:], [(45, 1)], 16, scale)
    out = M.paged_decode_attention_fp8(*(x.to(DEV) for x in (-q, kc, vc, sc, table)), kvl, 16, scale=scale)
    assert torch.isnan(out[0]).all()  # above it: as infinities are


# chunks whose rows fill the card's CTAs, and few rows, whose keys several CTAs share
SPANS = {"many rows": [(700, 700), (1, 1), (300, 200)], "few rows": [(2100, 20), (50, 3), (17, 1)]}


def prefill(q, kc, vc, sc, table, spans, bs, scale):
    rows, cached, qlen = (torch.tensor(x, device=DEV) for x in
                          (range(len(spans)), [n - r for n, r in spans], [r for _, r in spans]))
    return M.paged_prefill_attention_fp8(*(x.to(DEV) for x in (q, kc, vc, sc, table)), rows, cached, qlen, bs,
                                         scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("spans", list(SPANS))
def test_prefill(spans, name, heads):
    spans = SPANS[spans]
    q, kc, vc, sc, table, scale = case(name, spans, heads, 16)
    check(prefill(q, kc, vc, sc, table, spans, 16, scale), q, kc, vc, sc, table, spans, 16, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
def test_prefill_logits_that_overflow(heads):
    for spans in SPANS.values():
        q, kc, vc, sc, table, _ = case("negative", spans, heads, 16)
        scale, first = 2e37, spans[0][1]
        q[first:] *= 1e-33
        out = prefill(q, kc, vc, sc, table, spans, 16, scale)
        assert (out[:first] == 0).all()
        check(out[first:], q[first:], kc, vc, sc, table[1:], spans[1:], 16, scale)
        out = prefill(-q, kc, vc, sc, table, spans, 16, scale)
        assert torch.isnan(out[:first]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("last", [False, True])
def test_some_keys_overflow(last, heads):
    """160 positions whose logits are below float32's range, before or behind 140 that count."""
    n, rows = 300, 4
    q, kc, vc, sc, table, _ = case("negative", [(n, rows)], heads, 16)
    scale = 2e37
    kept = table[:, :9] if last else table[:, 10:]
    length = 144 if last else 140
    sc[kept[0], :, 0] *= 1e-33
    out = prefill(q, kc, vc, sc, table, [(n, rows)], 16, scale)
    one = M.paged_decode_attention_fp8(*(x.to(DEV) for x in (q[-1:], kc, vc, sc, table)),
                                       torch.tensor([n], dtype=torch.int32, device=DEV), 16, scale=scale)
    if last:  # every row attends all of what counts
        for r in range(rows):
            check(out[r:r + 1], q[r:r + 1], kc, vc, sc, kept, [(length, 1)], 16, scale)
    else:
        check(out, q, kc, vc, sc, kept, [(length, rows)], 16, scale)
    check(one, q[-1:], kc, vc, sc, kept, [(length, 1)], 16, scale)
