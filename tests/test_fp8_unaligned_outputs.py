"""Outputs of the 8-bit cache's operators whose rows are not 16-byte aligned: rows that a call leaves alone stay."""

from __future__ import annotations

import pytest
import torch

import mini_vllm_b200 as M
from mini_vllm_b200.attention import paged_attention_fp8 as P

E4M3 = torch.float8_e4m3fn
SHAPES = ["odd offset", "odd stride", "odd head stride"]


def room(kind, rows, heads, d, device, fill=5.0):
    """(all of the memory, a view [rows, heads, d] of it whose rows are not aligned)."""
    if kind == "odd offset":
        x = torch.full((rows * heads * d + 3,), fill, dtype=torch.bfloat16, device=device)
        return x, x[3:].view(rows, heads, d)
    if kind == "odd stride":
        x = torch.full((rows, heads * d + 4), fill, dtype=torch.bfloat16, device=device)
        return x, x[:, :heads * d].view(rows, heads, d)
    x = torch.full((rows, heads, d + 1), fill, dtype=torch.bfloat16, device=device)
    return x, x[..., :d]


@pytest.mark.parametrize("kind", SHAPES)
def test_what_the_kernel_writes_starts_as_the_output(kind):
    _, out = room(kind, 4, 3, 64, "cpu")
    out.copy_(torch.randn(4, 3, 64))
    got, target = P._output(out, torch.empty(4, 3, 64, dtype=torch.bfloat16), "out")
    assert got is out and P._aligned(target) and target.data_ptr() != out.data_ptr() and torch.equal(target, out)


def cache(num_blocks, kh, bs, d):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(0)
    codes = [torch.randn(num_blocks, kh, bs, d, generator=g, device=dev).mul(50).to(E4M3) for _ in range(2)]
    return (*codes, torch.full((num_blocks, kh, 2), 2.0 ** -6, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", SHAPES)
@pytest.mark.parametrize("cached,query", [([7, 40], [21, 60]), ([900, 3], [5, 2])])  # (shared keys in the second)
def test_prefill_rows_behind_the_last_chunk(kind, cached, query):
    dev = torch.device("cuda", 0)
    kv = cache(80, 2, 16, 64)
    table = torch.arange(80, device=dev)[None].expand(2, 80)
    used = sum(query)
    q = torch.randn(used + 9, 14, 64, device=dev).bfloat16()
    want = M.paged_prefill_attention_fp8(q, *kv, table, [0, 1], cached, query, 16)
    memory, out = room(kind, used + 9, 14, 64, dev)
    got = M.paged_prefill_attention_fp8(q, *kv, table, [0, 1], cached, query, 16, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:used], want[:used])
    out[:used] = 5.0
    assert (memory == 5.0).all()
    with pytest.raises(IndexError):  # more tokens than query has rows: nothing is written
        M.paged_prefill_attention_fp8(q, *kv, table, [0, 1], cached, [query[0], used + 20], 16, out=out)
    assert (memory == 5.0).all()
    M.check_device_errors(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", SHAPES)
def test_rotated_queries_of_bad_positions_stay(kind):
    dev = torch.device("cuda", 0)
    T, H, KH, D = 6, 14, 2, 64
    cos, sin = M.rope_tables(D, max_seq_len=32, dtype=torch.float32, device=dev)
    pos = torch.tensor([3, 40, 5, -1, 7, 31], device=dev)
    slots = torch.arange(T, device=dev)
    k, v = (torch.randn(T, KH, D, device=dev).bfloat16() for _ in range(2))
    start = torch.randn(T, H, D, device=dev).bfloat16()
    good = [0, 2, 4, 5]
    want, _ = M.rope_cache_write_fp8(start[good], k[good], v[good], pos[good], cos, sin, *cache(4, KH, 16, D),
                                     slots[good], 16)
    for in_place in (True, False):
        memory, out = room(kind, T, H, D, dev)
        if in_place:
            out.copy_(start)
        q = out if in_place else start
        with pytest.raises(IndexError, match="position"):
            M.rope_cache_write_fp8(q, k, v, pos, cos, sin, *cache(4, KH, 16, D), slots, 16, query_out=out)
        assert torch.equal(out[good], want)
        for t in (1, 3):
            assert torch.equal(out[t], start[t] if in_place else torch.full_like(start[t], 5.0))
        out.fill_(5.0)
        assert (memory == 5.0).all()
    M.check_device_errors(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", SHAPES)
def test_decode(kind):
    dev = torch.device("cuda", 0)
    kv = cache(20, 2, 16, 64)
    table = torch.arange(20, device=dev).view(2, 10)
    q = torch.randn(2, 14, 64, device=dev).bfloat16()
    lens = torch.tensor([150, 7], dtype=torch.int32, device=dev)
    memory, out = room(kind, 2, 14, 64, dev)
    M.paged_decode_attention_fp8(q, *kv, table, lens, 16, out=out)
    assert torch.equal(out, M.paged_decode_attention_fp8(q, *kv, table, lens, 16))
    out.fill_(5.0)
    assert (memory == 5.0).all()
