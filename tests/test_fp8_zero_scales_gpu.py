"""Attention behind blocks whose value scale is 0: the first scale above 0 is the unit of the values."""

from __future__ import annotations

import pytest
import torch

import mini_vllm_b200 as M
from test_fp8_cache_gpu import check_decode, check_prefill, decode_case, prefill_case

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def zero_first(sc, table, bs, positions):
    for b in range(-(-positions // bs)):
        sc[table[:, b], :, 1] = 0.0


@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("bs,positions", [(16, 64), (16, 150), (64, 64), (256, 256), (16, 600)])
@pytest.mark.parametrize("rows", [3, 700])
def test_prefill(rows, bs, positions, heads):
    """Scales that are all 2^-k times as large give the same bits 2^-k times as large."""
    cached, query = [1200], [rows]
    q, kc, vc, sc, table = prefill_case(5, cached, query, heads, bs, torch.bfloat16)
    zero_first(sc, table, bs, positions)
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], cached, query, bs)
    check_prefill(out, q, kc, vc, sc, table, cached, query, bs)
    for k in (15, 30, 60):
        small = sc.clone()
        small[..., 1] *= 2.0 ** -k
        got = M.paged_prefill_attention_fp8(q, kc, vc, small, table, [0], cached, query, bs)
        assert torch.equal(got.float() * 2.0 ** k, out.float())


@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("bs,positions", [(16, 16), (16, 150), (256, 256)])
def test_decode(bs, positions, heads):
    lens = [1200, 400]
    q, kc, vc, sc, table, kvl = decode_case(6, lens, heads, bs, torch.bfloat16)
    zero_first(sc, table, bs, positions)
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, bs)
    check_decode(out, q, kc, vc, sc, table, lens, bs)
    for k in (15, 30, 60):
        small = sc.clone()
        small[..., 1] *= 2.0 ** -k
        got = M.paged_decode_attention_fp8(q, kc, vc, small, table, kvl, bs)
        assert torch.equal(got.float() * 2.0 ** k, out.float())


@pytest.mark.parametrize("rows", [3, 700])
def test_nothing_but_zeros(rows):
    q, kc, vc, sc, table = prefill_case(7, [300], [rows], (14, 2, 64), 16, torch.float16)
    sc[..., 1] = 0.0
    assert (M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], [300], [rows], 16) == 0).all()
