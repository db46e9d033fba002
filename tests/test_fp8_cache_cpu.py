"""Refusals and host logic of the 8-bit cache's operators (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fp8_model as F
import mini_vllm_b200 as M
from mini_vllm_b200 import _native

E4M3 = torch.float8_e4m3fn


def cache(num_blocks=4, kh=2, bs=16, d=64, dtype=E4M3):
    return (torch.zeros(num_blocks, kh, bs, d, dtype=torch.uint8).view(E4M3).to(dtype) if dtype != E4M3
            else torch.zeros(num_blocks, kh, bs, d, dtype=torch.uint8).view(E4M3),
            torch.zeros(num_blocks, kh, bs, d, dtype=torch.uint8).view(E4M3), torch.zeros(num_blocks, kh, 2))


def write(kv=None, shape=(3, 2, 64), dtype=torch.bfloat16, slots=3, bs=16):
    kc, vc, sc = kv or cache()
    x = torch.zeros(shape, dtype=dtype)
    M.paged_cache_write_fp8(x, x, kc, vc, sc, torch.zeros(slots, dtype=torch.int64), bs)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=torch.float32), "bf16 or f16"),
    (dict(shape=(3, 128)), "num_tokens"),
    (dict(kv=cache(dtype=torch.bfloat16)), "float8_e4m3fn"),
    (dict(kv=cache(d=96), shape=(3, 2, 96)), "head_dim"),
    (dict(kv=cache(bs=8), bs=8), "power of 2"),
    (dict(kv=cache(bs=48), bs=48), "power of 2"),
    (dict(kv=cache(bs=2048), bs=2048), "power of 2"),
    (dict(bs=32), "dim2"),
    (dict(kv=cache()[:2] + (torch.zeros(4, 2),)), "kv_scale"),
    (dict(kv=cache()[:2] + (torch.zeros(4, 2, 2, dtype=torch.float16),)), "kv_scale"),
    (dict(kv=tuple(c.transpose(1, 2) for c in cache(kh=16)[:2]) + (torch.zeros(4, 16, 2),)), "contiguous"),
    (dict(), "CUDA device"),
])
def test_write_refusals(kw, match):
    with pytest.raises(AssertionError, match=match) as e:
        write(**kw)
    assert isinstance(e.value, ValueError)


def test_attention_refusals():
    kc, vc, sc = cache()
    bt, kvl = torch.zeros(1, 2, dtype=torch.int64), torch.ones(1, dtype=torch.int32)
    for q, match in ((torch.zeros(1, 14, 64), "bf16 or f16"), (torch.zeros(14, 64).bfloat16(), "query must be"),
                     (torch.zeros(1, 14, 64).bfloat16(), "CUDA device")):
        with pytest.raises(AssertionError, match=match):
            M.paged_decode_attention_fp8(q, kc, vc, sc, bt, kvl, 16)
        with pytest.raises(AssertionError, match=match):
            M.paged_prefill_attention_fp8(q, kc, vc, sc, bt, [0], [0], [1], 16)
    # the 16-bit functions do not take the 8-bit cache for theirs
    with pytest.raises(AssertionError):
        M.paged_decode_attention(torch.zeros(1, 14, 64).bfloat16(), kc, vc, bt, kvl, 16)
    with pytest.raises(AssertionError):
        M.paged_cache_write(torch.zeros(1, 2, 64).bfloat16(), torch.zeros(1, 2, 64).bfloat16(), kc, vc,
                            torch.zeros(1, dtype=torch.int64), 16)


def test_rope_refusals():
    kc, vc, sc = cache()
    x, q = torch.zeros(3, 2, 64).half(), torch.zeros(3, 14, 64).half()
    i = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(AssertionError, match="bf16 or f16"):
        M.rope_cache_write_fp8(q.float(), x.float(), x.float(), i, *M.rope_tables(64, max_seq_len=4), kc, vc, sc, i, 16)
    with pytest.raises(AssertionError, match="CUDA device"):
        M.rope_cache_write_fp8(q, x, x, i, *M.rope_tables(64, max_seq_len=4), kc, vc, sc, i, 16)


def test_library_checks_without_a_gpu():
    lib, n = _native.lib(), ctypes.c_int64()
    BF16 = _native.DTYPE_BF16

    def w(tokens, bs=16, d=64, dtype=BF16, ptr=None):
        return lib.mvb_kv_cache_write_fp8(ptr, 128, 64, ptr, 128, 64, ptr, ptr, ptr, ptr, tokens, 2, d, bs, 4, dtype,
                                          None, 0, ptr, None)

    assert w(0) == _native.OK and w(1) == _native.ERR_INVALID_ARG and w(-1) == _native.ERR_INVALID_ARG
    assert w(1, bs=8) == _native.ERR_BLOCK_SIZE and w(1, bs=24) == _native.ERR_BLOCK_SIZE
    assert w(1, d=32) == _native.ERR_HEAD_DIM and w(1, dtype=_native.DTYPE_F32) == _native.ERR_DTYPE
    assert w(1, ptr=8) == _native.ERR_ALIGNMENT and w(5000, ptr=4096) == _native.ERR_WORKSPACE
    assert lib.mvb_kv_cache_write_fp8_workspace(2048, 10, 16, ctypes.byref(n)) == _native.OK and n.value == 0
    assert lib.mvb_kv_cache_write_fp8_workspace(2049, 10, 16, ctypes.byref(n)) == _native.OK and n.value == 640
    assert lib.mvb_kv_cache_write_fp8_workspace(2049, 0, 16, ctypes.byref(n)) == _native.ERR_INVALID_ARG

    def d(seqs, heads=14, kv=2, dim=64, bs=16, maxb=8, dtype=BF16, ptr=None, ws=None, wsb=0):
        return lib.mvb_paged_decode_fp8(ptr, 64, 64, ptr, ptr, ptr, ptr, 8, maxb, ptr, ptr, 64, 64, seqs, heads, kv, dim,
                                        bs, 100, 0.1, dtype, ws, wsb, ptr, None)

    assert d(0) == _native.OK and d(1) == _native.ERR_INVALID_ARG and d(6145) == _native.ERR_INVALID_ARG
    assert d(1, heads=15) == _native.ERR_HEADS and d(1, dim=80) == _native.ERR_HEAD_DIM
    assert d(1, bs=8) == _native.ERR_BLOCK_SIZE and d(1, dtype=_native.DTYPE_F32) == _native.ERR_DTYPE
    assert d(1, ptr=4096, maxb=9) == _native.ERR_INVALID_ARG  # the table's rows are shorter
    assert d(1, ptr=8) == _native.ERR_ALIGNMENT and d(1, ptr=4096) == _native.ERR_WORKSPACE
    assert d(6144, maxb=1 << 26) == _native.ERR_INVALID_ARG  # tile numbers are 32-bit
    assert lib.mvb_paged_decode_fp8_workspace(256, 14, 2, 64, 16, 100, 128, BF16, ctypes.byref(n)) == _native.OK
    assert n.value >= 148 * 2 * (16 + 8 * 66 * 4)

    def p(chunks, total, heads=14, kv=2, dim=64, bs=16, dtype=BF16, ptr=None, maxb=8, ws=None, size=0):
        return lib.mvb_paged_prefill_fp8(ptr, 64, 64, ptr, ptr, ptr, ptr, 4, 1000, maxb, ptr, ptr, ptr, chunks, total,
                                         ptr, 64, 64, heads, kv, dim, bs, 100, 0.1, dtype, ws, size, ptr, None)

    assert p(0, 5) == _native.OK and p(1, 0) == _native.OK and p(1, 1) == _native.ERR_INVALID_ARG
    assert p(4097, 5000) == _native.ERR_INVALID_ARG and p(1, 1, heads=15) == _native.ERR_HEADS
    assert p(1, 1, dim=32) == _native.ERR_HEAD_DIM and p(1, 1, bs=8) == _native.ERR_BLOCK_SIZE
    assert p(1, 1, dtype=_native.DTYPE_F32) == _native.ERR_DTYPE and p(1, 1, ptr=8) == _native.ERR_ALIGNMENT
    # few rows after many keys: a workspace
    assert p(1, 5, ptr=4096, maxb=100) == p(1, 5, ptr=4096, maxb=100, ws=4096, size=64) == _native.ERR_WORKSPACE
    assert p(1, 5, ptr=4096, maxb=100, ws=4096 + 16, size=1 << 30) == _native.ERR_WORKSPACE
    w = lambda *c: (lib.mvb_paged_prefill_fp8_workspace(*c, ctypes.byref(n)), n.value)  # noqa: E731
    assert w(1, 5, 14, 2, 64, 16, 100) == (_native.OK, 12 * 5 * 14 * 65 * 4)  # 25 steps of 64 keys: twelve shares of two or more
    assert w(1, 5, 14, 2, 64, 16, 12) == w(30, 8192, 14, 2, 64, 16, 1000) == w(0, 0, 14, 2, 64, 16, 0) == (_native.OK, 0)
    assert w(1, 5, 15, 2, 64, 16, 1)[0] == _native.ERR_HEADS and w(1, 5, 14, 2, 96, 16, 1)[0] == _native.ERR_HEAD_DIM
    assert w(1, 1 << 28, 14, 2, 64, 16, 1)[0] == w(1, 1, 14, 2, 64, 1024, 1 << 20)[0] == _native.ERR_INVALID_ARG


def test_pool_of_8_bits():
    pool = M.KVCachePool.allocate(2, 16, 32, 4, 128, E4M3, torch.device("cpu"))
    assert [tuple(s.shape) for s in pool.kv_scales] == [(16, 4, 2)] * 2 and (pool.kv_scales[0] == 0).all()
    assert pool.bytes_per_block_per_layer == 2 * 4 * 32 * 128 + 4 * 8
    pool.kv_scales[1].fill_(3.0)
    pool.reset()
    assert (pool.kv_scales[1] == 0).all() and (pool.key_caches[0].view(torch.uint8) == 0).all()
    assert M.KVCachePool.allocate(1, 16, 16, 2, 64, torch.bfloat16, torch.device("cpu")).kv_scales is None


def test_model_codes():
    """The model's rounding against torch's own conversion, over every tie and neighbour."""
    grid = torch.arange(127, dtype=torch.uint8).view(E4M3).float()
    mid = (grid[1:] + grid[:-1]) / 2
    x = torch.cat([grid, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), torch.linspace(-448, 448, 10001)])
    x = torch.cat([x, -x])
    assert torch.equal(F.to_codes(x.double()), x.to(E4M3).view(torch.uint8))
    for e in (-30, 0, 5):
        assert F.scale_for(448.0 * 2.0 ** e) == 2.0 ** e and F.scale_for(448.0 * 2.0 ** e * (1 + 2.0 ** -23)) == 2.0 ** (e + 1)
    assert F.scale_for(0.0) == 2.0 ** -100
