"""The 8-bit KV cache on the GPU: writes, decode and prefill against the model in 64 bits (tests/fp8_model.py)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import fp8_model as F
import mini_vllm_b200 as M
from mini_vllm_b200 import _native

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
E4M3 = torch.float8_e4m3fn
HEADS = [(14, 2, 64), (32, 8, 128), (5, 5, 64), (16, 1, 128), (24, 2, 64), (40, 2, 128)]


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def bits(t):
    return t.view(torch.uint8)


def make_cache(g, num_blocks, kh, bs, d, spread=1.0):
    """Codes of normal values under power-of-two scales."""
    caches, scales = [], []
    for _ in range(2):
        x = torch.randn(num_blocks, kh, bs, d, generator=g, device=DEV) * torch.exp(
            spread * torch.randn(num_blocks, kh, 1, 1, generator=g, device=DEV))
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448.0)))
        caches.append((x / s[..., None, None]).to(E4M3))
        scales.append(s)
    return caches[0], caches[1], torch.stack(scales, -1).contiguous()


def make_tables(seed, lens, bs, extra=3):
    """Block tables for sequences of `lens` tokens, -1 padded, from a permuted pool."""
    r = np.random.RandomState(seed)
    need = [-(-n // bs) for n in lens]
    num_blocks = sum(need) + extra
    perm = r.permutation(num_blocks)
    table = np.full((len(lens), max(max(need), 1)), -1, dtype=np.int64)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    return torch.from_numpy(table).to(DEV), num_blocks


def poison(cache, table, lens, bs):
    """NaN codes in every slot of the tables' blocks behind the last token."""
    for i, n in enumerate(lens):
        if n > 0 and n % bs:
            bits(cache)[table[i, n // bs], :, n % bs:] = 0x7F


# ---------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------
def write_case(g, tokens, heads, dtype, table_dtype, rows=512):
    H, KH, D = heads
    qkv = torch.randn(tokens, H + 2 * KH, D, generator=g, device=DEV)
    qkv *= torch.exp(1.5 * torch.randn(tokens, H + 2 * KH, 1, generator=g, device=DEV))
    qkv = qkv.to(dtype)
    pos = torch.randint(0, rows, (tokens,), generator=g, device=DEV)
    cos, sin = M.rope_tables(D, max_seq_len=rows, dtype=table_dtype, device=DEV)
    return qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:], pos, cos, sin


def check_write(heads, bs, dtype, table_dtype, slots, num_blocks, seed=0, calls=1):
    """`calls` writes into one cache, each of new rows into `slots`; scales and value codes are compared bit for bit.

    A rotated row is a product and a fused multiply-add in float32: off by at most 2^-24 (|y s| + |r|) from
    the exact rotation, |r| <= |x c| + |y s|.  Rounded to 16 bits it is half a step more; coded, it can take the
    other neighbour where the exact value is that near a tie, which of 2^19 float32 values between two ties is
    about one in 2^18: at most `cells` / 2^18 expected, and 8 more allowed.  Scales are those of exact sums."""
    g = gen(seed)
    H, KH, D = heads
    kc, vc, sc = make_cache(g, num_blocks, KH, bs, D)
    slots = torch.as_tensor(slots, dtype=torch.int64, device=DEV)
    mk, mv, ms = kc.cpu(), vc.cpu(), sc.cpu()
    for _ in range(calls):
        q, k, v, pos, cos, sin = write_case(g, len(slots), heads, dtype, table_dtype)
        qo, ko = M.rope_cache_write_fp8(q, k, v, pos, cos, sin, kc, vc, sc, slots, bs, return_key=True)
        rq, rk = (F.rotate(x, cos, sin, pos) for x in (q, k))
        for got, ref, x in ((qo, rq, q), (ko, rk, k)):
            ref, terms = ref.double(), F.rotate(x.abs(), cos.abs(), -sin.abs(), pos).abs().double()
            terms = torch.maximum(terms, F.rotate(x.abs(), cos.abs(), sin.abs(), pos).abs().double())
            limit = F.UNIT[dtype] * ref.abs() + 2.0 ** -22 * terms + 2.0 ** -25
            assert ((got.double() - ref).abs() <= limit).all()
        F.write(rk.cpu(), v.float().cpu(), mk, mv, ms, slots.cpu(), bs)
        assert torch.equal(sc.cpu(), ms) and torch.equal(bits(vc).cpu(), bits(mv))
        apart = bits(kc).cpu() != bits(mk)
        assert apart.sum() <= k.numel() / 2 ** 18 + 8
        a, b = kc.cpu()[apart.view(mk.shape)].float(), mk[apart.view(mk.shape)].float()
        assert ((a - b).abs() <= torch.maximum(a.abs() / 8, torch.tensor(2.0 ** -9))).all()  # neighbours
        mk = kc.cpu()


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype,table", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                         (torch.bfloat16, torch.bfloat16)])
def test_write_ragged_chunks(heads, dtype, table):
    # pieces of four blocks: a block's middle, its start, all of it, its last slot
    slots = list(range(5, 12)) + list(range(16, 17)) + list(range(48, 64)) + [47, -1, 79]
    check_write(heads, 16, dtype, table, slots, 6, calls=2)


@pytest.mark.parametrize("bs", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_write_block_sizes_and_orders(bs, tokens):
    r = np.random.RandomState(bs + tokens)
    num_blocks = max(3, 2 * tokens // bs)
    slots = r.permutation(num_blocks * bs)[:tokens]  # any order, any block
    slots[r.rand(tokens) < 0.1] = -1
    check_write((14, 2, 64), bs, torch.bfloat16, torch.float32, slots, num_blocks, calls=2)


@pytest.mark.parametrize("shuffled", [False, True])
def test_write_many_tokens(shuffled):
    """Past the size up to which a token's CTA looks at every slot (2048)."""
    r = np.random.RandomState(3)
    slots = np.concatenate([np.arange(7, 1900), np.arange(2048, 2500), np.full(9, -1)])
    if shuffled:
        r.shuffle(slots)
    check_write((14, 2, 64), 16, torch.bfloat16, torch.float32, slots, 160, calls=2)
    check_write((8, 8, 128), 64, torch.float16, torch.float16, slots, 40, calls=2)


def test_write_token_by_token_is_the_write_at_once():
    """Powers of two: codes that are normal (2^-6 and up) do not depend on how a block was filled."""
    g = gen(1)
    KH, D, bs, T = 2, 64, 16, 40
    k = (torch.randn(T, KH, D, generator=g, device=DEV) * torch.exp(torch.randn(T, KH, 1, generator=g, device=DEV)))
    k, v = k.bfloat16(), torch.randn(T, KH, D, generator=g, device=DEV).bfloat16()
    at_once, steps = (make_cache(gen(2), 4, KH, bs, D) for _ in range(2))
    slots = torch.arange(T, device=DEV)
    M.paged_cache_write_fp8(k, v, *at_once, slots, bs)
    for t in range(T):
        M.paged_cache_write_fp8(k[t:t + 1], v[t:t + 1], *steps, slots[t:t + 1], bs)
    assert torch.equal(at_once[2][:3], steps[2][:3])
    for a, b in zip(at_once[:2], steps[:2]):
        x, y = (c.float().transpose(1, 2).reshape(-1, KH, D)[:T] for c in (a, b))
        normal = x.abs() >= 2.0 ** -6
        assert torch.equal(x[normal], y[normal])
        assert ((x - y).abs() <= 2.0 ** -9).all()  # two roundings below: a step at most


def test_write_zeros_infinities_and_nan():
    bs, KH, D = 16, 2, 64
    kc, vc, sc = make_cache(gen(4), 3, KH, bs, D)
    sc[1] = torch.tensor([0.0, math.nan], device=DEV)  # never written: no scale yet
    k = torch.zeros(4, KH, D, device=DEV)
    v = torch.ones(4, KH, D, device=DEV)
    k[1, 0, 3], k[1, 0, 4], k[1, 0, 5] = math.inf, -math.inf, math.nan
    v[2, 1, 7] = 3e38
    slots = torch.tensor([0, 1, 2, 20], device=DEV)
    mk, mv, ms = kc.cpu(), vc.cpu(), sc.cpu()
    k, v = k.bfloat16(), v.bfloat16()
    M.paged_cache_write_fp8(k, v, kc, vc, sc, slots, bs)
    F.write(k.float().cpu(), v.float().cpu(), mk, mv, ms, slots.cpu(), bs)
    assert torch.equal(sc.cpu(), ms) and torch.equal(bits(kc).cpu(), bits(mk)) and torch.equal(bits(vc).cpu(), bits(mv))
    assert sc[0, 0, 0] == 2.0 ** -100 and torch.isnan(kc.float()[0, 0, 1, 5])
    assert kc.float()[0, 0, 1, 3] == 448 and kc.float()[0, 0, 1, 4] == -448


@pytest.mark.parametrize("tokens", [1, 700, 2200])
def test_write_one_row_per_block(tokens):
    """A decode step: every block has one new row, in any place."""
    r = np.random.RandomState(tokens)
    slots = r.permutation(tokens) * 16 + r.randint(0, 16, tokens)
    check_write((32, 8, 128), 16, torch.bfloat16, torch.bfloat16, slots, tokens, calls=2)


def test_write_border_of_a_scale():
    """448 * 2^k keeps its scale, the next float32 above takes the next one."""
    bs, KH, D = 16, 1, 64
    for x, s in ((448.0, 1.0), (449.0, 2.0), (1.75, 2.0 ** -8), (1.7578125, 2.0 ** -7), (2.0 ** -20, 2.0 ** -28)):
        kc, vc, sc = make_cache(gen(5), 1, KH, bs, D)
        k = torch.full((1, KH, D), x, device=DEV).half()
        assert float(k[0, 0, 0]) == x  # exact in f16
        M.paged_cache_write_fp8(k, k, kc, vc, sc, torch.zeros(1, dtype=torch.int64, device=DEV), bs)
        assert float(sc[0, 0, 0]) == F.scale_for(x) == s


def test_write_strides_in_place_and_other_dtypes_of_indices():
    g = gen(6)
    H, KH, D, bs, T = 14, 2, 64, 16, 21
    q, k, v, pos, cos, sin = write_case(g, T, (H, KH, D), torch.bfloat16, torch.float32)
    slots = torch.arange(T, device=DEV)
    ref = make_cache(gen(7), 4, KH, bs, D)
    qo, _ = M.rope_cache_write_fp8(q, k, v, pos, cos, sin, *ref, slots, bs)
    for change in ("transposed", "odd", "in place", "int32", "strided out"):
        got = make_cache(gen(7), 4, KH, bs, D)
        a, b, c = q.clone(), k.clone(), v.clone()
        kw, p, s = {}, pos, slots
        if change == "transposed":
            b = k.transpose(1, 2).contiguous().transpose(1, 2)  # last dimension not contiguous
        elif change == "odd":
            room = torch.empty(T, KH, D + 1, dtype=k.dtype, device=DEV)
            room[..., 1:] = v
            c = room[..., 1:]  # rows at odd addresses
        elif change == "in place":
            kw = {"query_out": a}
        elif change == "int32":
            p, s = pos.int(), slots.int().cpu()
        else:
            kw = {"query_out": torch.empty(T, H, D + 3, dtype=q.dtype, device=DEV)[..., 2:D + 2]}
        out, _ = M.rope_cache_write_fp8(a, b, c, p, cos, sin, *got, s, bs, **kw)
        assert torch.equal(out, qo), change
        assert all(torch.equal(bits(x), bits(y)) for x, y in zip(got, ref)), change
        if kw:
            assert out.data_ptr() == kw["query_out"].data_ptr()


def test_write_device_errors():
    bs, KH, D = 16, 2, 64
    for many in (False, True):
        n = 2100 if many else 3
        cache = make_cache(gen(8), 100, KH, bs, D)
        k = torch.ones(n, KH, D, device=DEV).half()
        slots = torch.full((n,), -1, dtype=torch.int64, device=DEV)
        slots[:3] = torch.tensor([5, 7, 5], device=DEV)
        with pytest.raises(AssertionError, match="Duplicate"):
            M.paged_cache_write_fp8(k, k, *cache, slots, bs)
        for bad in (1600, -2, 1 << 40):
            before = [c.clone() for c in cache]
            slots[:3] = torch.tensor([bad, -1, -1], device=DEV)
            with pytest.raises(IndexError, match="out of range"):
                M.paged_cache_write_fp8(k, k, *cache, slots, bs)
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(cache, before))
        slots[:3] = torch.tensor([17, 18, 33], device=DEV)
        pos = torch.zeros(n, dtype=torch.int64, device=DEV)
        pos[1] = 64
        cos, sin = M.rope_tables(D, max_seq_len=64, device=DEV)
        before = [c.clone() for c in cache]
        with pytest.raises(IndexError, match="position"):
            M.rope_cache_write_fp8(k, k, k, pos, cos, sin, *cache, slots, bs)
        assert torch.equal(bits(cache[0])[1, :, 2], bits(before[0])[1, :, 2])  # the token with the bad position
        assert (cache[0].float()[2, :, 1] * cache[2][2, :, :1] == 1).all()     # the others are written
        M.check_device_errors(DEV)


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def decode_case(seed, lens, heads, bs, dtype, qscale=1.0, spread=1.0):
    g = gen(seed)
    H, KH, D = heads
    table, num_blocks = make_tables(seed, lens, bs)
    kc, vc, sc = make_cache(g, num_blocks, KH, bs, D, spread)
    for c in (kc, vc):
        poison(c, table, lens, bs)
    q = (torch.randn(len(lens), H, D, generator=g, device=DEV) * qscale).to(dtype)
    return q, kc, vc, sc, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def check_decode(out, q, kc, vc, sc, table, lens, bs, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for i, n in enumerate(lens):
        blocks = table[i, :-(-n // bs)]
        k, v = F.dequant(kc, sc, 0, blocks, n), F.dequant(vc, sc, 1, blocks, n)
        F.check(out[i:i + 1], *F.attend(q[i:i + 1], k, v, n, scale))


LENS = {"one": [1], "short": [1, 15, 16, 17, 31, 2, 48], "mixed": [700, 1, 33, 2048, 129, 5, 64, 1000],
        "long": [5000], "many": list(range(1, 180)), "few long": [3333, 4097, 2]}


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode(lens, heads, dtype):
    lens = LENS[lens]
    q, kc, vc, sc, table, kvl = decode_case(len(lens), lens, heads, 16, dtype)
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    check_decode(out, q, kc, vc, sc, table, lens, 16)


@pytest.mark.parametrize("bs", [32, 64, 128, 1024])
def test_decode_block_sizes(bs):
    lens = LENS["mixed"]
    q, kc, vc, sc, table, kvl = decode_case(bs, lens, (14, 2, 64), bs, torch.bfloat16)
    check_decode(M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, bs), q, kc, vc, sc, table, lens, bs)


@pytest.mark.parametrize("dtype,qscale", [(torch.bfloat16, 1e-30), (torch.bfloat16, 8.0), (torch.float16, 8.0),
                                          (torch.float16, 1e-4), (torch.bfloat16, 0.0)])
def test_decode_query_range(dtype, qscale):
    lens = [77, 300]
    q, kc, vc, sc, table, kvl = decode_case(11, lens, (14, 2, 64), 16, dtype, qscale, spread=0.3)
    check_decode(M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16), q, kc, vc, sc, table, lens, 16)


def test_decode_large_queries_and_small_scales():
    """Logits stay moderate while the query is beyond f16 and the keys' scales tiny; scales need not be powers of two."""
    lens = [90, 513]
    q, kc, vc, sc, table, kvl = decode_case(12, lens, (32, 8, 128), 16, torch.bfloat16, 1e20)
    sc[..., 0] *= 1.3e-20
    sc[..., 1] *= 0.7
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16, scale=0.05)
    check_decode(out, q, kc, vc, sc, table, lens, 16, scale=0.05)


def test_decode_rising_logits():
    """The running maximum moves at every tile: keys in the query's direction, longer from token to token."""
    H, KH, D, bs, n = 14, 2, 64, 16, 400
    q, kc, vc, sc, table, kvl = decode_case(13, [n], (H, KH, D), bs, torch.float16)
    up = torch.linspace(0.1, 3.0, n, device=DEV)
    k = q[0, ::7][None] * up[:, None, None]
    slots = table[0].repeat_interleave(bs)[:n] * bs + torch.arange(n, device=DEV) % bs
    M.paged_cache_write_fp8(k.half(), torch.randn(n, KH, D, generator=gen(1), device=DEV).half(), kc, vc, sc, slots, bs)
    check_decode(M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, bs), q, kc, vc, sc, table, [n], bs)


def test_decode_same_bits_every_time_and_out():
    lens = LENS["mixed"] * 20
    q, kc, vc, sc, table, kvl = decode_case(14, lens, (14, 2, 64), 16, torch.bfloat16)
    a = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    room = torch.full((len(lens) + 2, 14, 80), 7.0, dtype=q.dtype, device=DEV)
    view = room[1:-1, :, 8:72]
    for _ in range(3):
        b = M.paged_decode_attention_fp8(q, kc, vc, sc, table.int(), kvl.long(), 16, out=view, strict=False)
        assert b.data_ptr() == view.data_ptr() and torch.equal(a, b)
    odd = torch.empty(len(lens), 14, 67, dtype=q.dtype, device=DEV)[..., 3:]
    assert torch.equal(M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16, out=odd), a) and torch.equal(odd, a)
    room[1:-1, :, 8:72] = 7.0
    assert (room == 7.0).all()  # nothing beside the output was written
    M.check_device_errors(DEV)


def test_decode_errors():
    lens = [40, 20, 64]
    q, kc, vc, sc, table, kvl = decode_case(15, lens, (14, 2, 64), 16, torch.bfloat16)
    kvl[1] = 0
    with pytest.raises(ValueError, match="kv_len_after"):
        M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16, strict=False)
    assert (out[1] == 0).all()
    check_decode(out[::2], q[::2], kc, vc, sc, table[::2], lens[::2], 16)
    with pytest.raises(ValueError):
        M.check_device_errors(DEV)
    kvl[1] = 65
    with pytest.raises(IndexError, match="insufficient"):
        M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    kvl[1] = 20
    for bad in (-1, kc.shape[0], 1 << 40):
        t = table.clone()
        t[1, 1] = bad
        with pytest.raises(IndexError, match="block_table entry"):
            M.paged_decode_attention_fp8(q, kc, vc, sc, t, kvl, 16)
        out = M.paged_decode_attention_fp8(q, kc, vc, sc, t, kvl, 16, strict=False)
        check_decode(out[1:2], q[1:2], kc, vc, sc, t[1:2], [16], 16)  # the bad block's tokens are left out
        with pytest.raises(IndexError):
            M.check_device_errors(DEV)
    t = torch.full_like(table, -1)
    assert (M.paged_decode_attention_fp8(q, kc, vc, sc, t, kvl, 16, strict=False) == 0).all()
    with pytest.raises(IndexError):
        M.check_device_errors(DEV)


def test_decode_far_into_a_large_cache():
    """Byte offsets past 2^32."""
    H, KH, D, bs = 16, 8, 128, 16
    num_blocks = (1 << 32) // (KH * bs * D) + 100
    g = gen(16)
    kc = torch.zeros(num_blocks, KH, bs, D, dtype=torch.uint8, device=DEV).view(E4M3)
    vc = torch.zeros(num_blocks, KH, bs, D, dtype=torch.uint8, device=DEV).view(E4M3)
    sc = torch.zeros(num_blocks, KH, 2, device=DEV)
    n = 150
    table = torch.arange(num_blocks - 10, num_blocks, device=DEV)[None]
    slots = (num_blocks - 10) * bs + torch.arange(n, device=DEV)
    k, v = (torch.randn(n, KH, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    M.paged_cache_write_fp8(k, v, kc, vc, sc, slots, bs)
    q = torch.randn(1, H, D, generator=g, device=DEV).bfloat16()
    kvl = torch.tensor([n], dtype=torch.int32, device=DEV)
    check_decode(M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, bs), q, kc, vc, sc, table, [n], bs)
    assert F.dequant(kc, sc, 0, table[0], n).sub(k.double().transpose(0, 1)).abs().max() < 0.3
    rows, cached = torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor([n - 1], device=DEV)
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, rows, cached, rows + 1, bs)
    check_decode(out, q, kc, vc, sc, table, [n], bs)


def test_decode_many_sequences():
    lens = [1 + i % 19 for i in range(6144)]
    q, kc, vc, sc, table, kvl = decode_case(17, lens, (4, 1, 64), 16, torch.float16)
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    pick = list(range(0, 6144, 401)) + [6143]
    check_decode(out[pick], q[pick], kc, vc, sc, table[pick], [lens[i] for i in pick], 16)
    with pytest.raises(AssertionError):
        M.paged_decode_attention_fp8(*(torch.cat([x, x[:1]]) if x is q else x for x in (q, kc, vc, sc)),
                                     torch.cat([table, table[:1]]), torch.cat([kvl, kvl[:1]]), 16)


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------
def prefill_case(seed, cached, query, heads, bs, dtype, spare=0):
    g = gen(seed)
    H, KH, D = heads
    lens = [c + q for c, q in zip(cached, query)]
    table, num_blocks = make_tables(seed, lens, bs)
    kc, vc, sc = make_cache(g, num_blocks, KH, bs, D)
    for c in (kc, vc):
        poison(c, table, lens, bs)
    q = torch.randn(sum(query) + spare, H, D, generator=g, device=DEV).to(dtype)
    return q, kc, vc, sc, table


def check_prefill(out, q, kc, vc, sc, table, cached, query, bs, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    at = 0
    for i, (c, n) in enumerate(zip(cached, query)):
        if n == 0:
            continue
        blocks = table[i, :-(-(c + n) // bs)]
        k, v = F.dequant(kc, sc, 0, blocks, c + n), F.dequant(vc, sc, 1, blocks, c + n)
        F.check(out[at:at + n], *F.attend(q[at:at + n], k, v, c + 1, scale))
        at += n


CHUNKS = {"one token": ([0], [1]), "one after many": ([1000], [1]), "first": ([0], [333]), "odd": ([77], [130]),
          "batch": ([0, 5, 129, 300, 16], [17, 1, 128, 65, 200]), "with empty": ([10, 3, 20], [5, 0, 40]),
          "long": ([900], [700])}


@pytest.mark.parametrize("chunks", list(CHUNKS))
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill(chunks, heads, dtype):
    cached, query = CHUNKS[chunks]
    q, kc, vc, sc, table = prefill_case(1, cached, query, heads, 16, dtype)
    n = len(cached)
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, list(range(n)), cached, query, 16)
    check_prefill(out, q, kc, vc, sc, table, cached, query, 16)


@pytest.mark.parametrize("bs", [32, 64, 128, 1024])
def test_prefill_block_sizes(bs):
    cached, query = CHUNKS["batch"]
    q, kc, vc, sc, table = prefill_case(bs, cached, query, (14, 2, 64), bs, torch.bfloat16)
    rows, c, n = (torch.tensor(x, device=DEV) for x in (range(5), cached, query))
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, rows, c, n, bs)
    check_prefill(out, q, kc, vc, sc, table, cached, query, bs)


def test_prefill_rows_behind_the_last_chunk_stay():
    cached, query = [7, 40], [21, 60]
    q, kc, vc, sc, table = prefill_case(2, cached, query, (14, 2, 64), 16, torch.bfloat16, spare=50)
    room = torch.full((131, 14, 80), 5.0, dtype=q.dtype, device=DEV)
    out = room[:, :, 8:72]
    got = M.paged_prefill_attention_fp8(q, kc, vc, sc, table.flip(0), [1, 0], cached, query, 16, out=out, scale=0.2)
    check_prefill(got[:81], q, kc, vc, sc, table, cached, query, 16, scale=0.2)
    out[:81] = 5.0
    assert (room == 5.0).all()


def test_prefill_rising_and_falling_logits():
    """Maxima that jump and masked keys that are far larger than the ones a row attends."""
    H, KH, D, bs, n = 14, 2, 64, 16, 500
    q, kc, vc, sc, table = prefill_case(3, [0], [n], (H, KH, D), bs, torch.float16)
    k = q[:, ::7] * torch.linspace(0.1, 4.0, n, device=DEV)[:, None, None]
    slots = table[0].repeat_interleave(bs)[:n] * bs + torch.arange(n, device=DEV) % bs
    for order in (slots, slots.flip(0)):
        kc2, vc2, sc2 = kc.clone(), vc.clone(), sc.clone()
        M.paged_cache_write_fp8(k.half(), torch.randn(n, KH, D, generator=gen(1), device=DEV).half(), kc2, vc2, sc2, order, bs)
        out = M.paged_prefill_attention_fp8(q, kc2, vc2, sc2, table, [0], [0], [n], bs)
        check_prefill(out, q, kc2, vc2, sc2, table, [0], [n], bs)


def test_prefill_query_range_and_scales():
    cached, query = [30], [200]
    q, kc, vc, sc, table = prefill_case(4, cached, query, (32, 8, 128), 16, torch.bfloat16)
    q *= 1e20
    sc[..., 0] *= 1.3e-20
    sc[..., 1] *= 0.7
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], cached, query, 16, scale=0.05)
    check_prefill(out, q, kc, vc, sc, table, cached, query, 16, scale=0.05)


def test_prefill_errors():
    cached, query = [30, 10], [40, 20]
    q, kc, vc, sc, table = prefill_case(5, cached, query, (14, 2, 64), 16, torch.bfloat16)
    call = lambda *a, **kw: M.paged_prefill_attention_fp8(q, kc, vc, sc, *a, 16, **kw)  # noqa: E731
    with pytest.raises(IndexError, match="insufficient"):
        call(table, [0, 1], [50, 10], query)
    out = call(table, [0, 1], [50, 10], query, strict=False)
    assert (out[:40] == 0).all()
    check_prefill(out[40:], q[40:], kc, vc, sc, table[1:], cached[1:], query[1:], 16)
    with pytest.raises(IndexError):
        M.check_device_errors(DEV)
    with pytest.raises(IndexError):
        call(table, [0, 2], cached, query)
    with pytest.raises(IndexError):
        call(table, [0, 1], [-1, 10], query)
    with pytest.raises(IndexError):
        call(table, [0, 1], cached, [40, 21])  # more tokens than query has rows
    t = table.clone()
    t[1, 0] = -1
    with pytest.raises(IndexError, match="block_table entry"):
        call(t, [0, 1], cached, query)
    M.check_device_errors(DEV)


# ---------------------------------------------------------------------------
# streams, graphs, and a run of all of it
# ---------------------------------------------------------------------------
def test_captured_calls_and_two_streams():
    lens = LENS["mixed"] * 8
    cases = [decode_case(s, lens, (14, 2, 64), 16, torch.bfloat16) for s in (20, 21)]
    want = [M.paged_decode_attention_fp8(*c, 16) for c in cases]
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(M.paged_decode_attention_fp8(*c, 16, strict=False))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):  # both at once, and an eager call between
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = M.paged_decode_attention_fp8(*cases[0], 16, strict=False)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(eager, want[0])
    got = []
    for s, c in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append(M.paged_decode_attention_fp8(*c, 16, strict=False))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_writes_with_new_rows():
    """A captured write replayed with other rows, slots and positions in the same tensors; many tokens too."""
    for T in (30, 2500):
        g = gen(22)
        bs, heads = 16, (14, 2, 64)
        num_blocks = 2 * T // bs + 2
        q, k, v, pos, cos, sin = write_case(g, T, heads, torch.bfloat16, torch.float32)
        q, k, v = q.clone(), k.clone(), v.clone()
        slots = torch.arange(T, device=DEV)
        a, b = (make_cache(gen(23), num_blocks, heads[1], bs, heads[2]) for _ in range(2))
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            qo, _ = M.rope_cache_write_fp8(q, k, v, pos, cos, sin, *a, slots, bs, strict=False)
        for i in range(3):
            q2, k2, v2, pos2, _, _ = write_case(g, T, heads, torch.bfloat16, torch.float32)
            order = torch.randperm(num_blocks * bs, generator=g, device=DEV)[:T] if i < 2 else torch.arange(3, T + 3, device=DEV)
            for dst, src in ((q, q2), (k, k2), (v, v2), (pos, pos2), (slots, order)):
                dst.copy_(src)
            graph.replay()
            want, _ = M.rope_cache_write_fp8(q2, k2, v2, pos2, cos, sin, *b, order, bs)
            assert torch.equal(qo, want) and all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))
        M.check_device_errors(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_backend_serves_from_an_8_bit_pool(dtype):
    """Prefill in two chunks, then decode steps, through the backend's methods: every output against the model
    on what the pool holds, and the pool against the model of the writes."""
    H, KH, D, bs, layers = 14, 2, 64, 16, 2
    backend = M.AttentionBackend.create(M.ModelConfig(num_heads=H, num_kv_heads=KH, head_dim=D), "b200")
    pool = backend.allocate_pool(layers, 24, bs, KH, D, E4M3, DEV)
    assert pool.kv_scales is not None and pool.bytes_per_block_per_layer == 2 * KH * bs * D + 8 * KH
    for kc, vc in zip(pool.key_caches, pool.value_caches):  # what the memory held
        bits(kc).fill_(0x7F)
        bits(vc).fill_(0x7F)
    model = [[c.cpu().clone() for c in (k, v, s)]
             for k, v, s in zip(pool.key_caches, pool.value_caches, pool.kv_scales)]
    table = torch.from_numpy(np.random.RandomState(0).permutation(24)[:14].reshape(2, 7)).to(DEV)
    g = gen(30)
    length = [0, 0]

    def rows(n, heads):
        return torch.randn(n, heads, D, generator=g, device=DEV).to(dtype)

    def step(new, kind):
        before = torch.tensor(length, device=DEV)
        n = torch.tensor(new, device=DEV)
        group = M.AttentionGroup([0, 1], kind, before, n, (before + n).to(torch.int64))
        meta = M.AttentionMetadata(groups=[group], block_size=bs, num_kv_heads=KH, head_dim=D)
        meta.prefill_block_tables = meta.decode_block_tables = table
        pos = [length[i] + j for i in (0, 1) for j in range(new[i])]
        seq = [i for i in (0, 1) for _ in range(new[i])]
        slots = torch.tensor([int(table[s, p // bs]) * bs + p % bs for s, p in zip(seq, pos)], device=DEV)
        T = len(pos)
        for layer in range(layers):
            q, k, v = rows(T, H), rows(T, KH), rows(T, KH)
            backend.write_kv_cache(layer, k, v, slots)
            F.write(k.float().cpu(), v.float().cpu(), *model[layer], slots.cpu(), bs)
            kc, vc, sc = pool.key_caches[layer], pool.value_caches[layer], pool.kv_scales[layer]
            for a, b in zip((kc, vc, sc), model[layer]):
                assert torch.equal(bits(a).cpu(), bits(b))
            if kind == "prefill_gpu":
                out = backend.prefill_attention(layer, q, k, v, meta, pool)
                check_prefill(out, q, kc, vc, sc, table, list(length), new, bs)
            else:
                out = backend.decode_attention(layer, q, meta, pool)
                check_decode(out, q, kc, vc, sc, table, [a + b for a, b in zip(length, new)], bs)
        for i in (0, 1):
            length[i] += new[i]

    step([19, 40], "prefill_gpu")
    step([30, 5], "prefill_gpu")
    for _ in range(20):
        step([1, 1], "decode_gpu")
    with pytest.raises(AssertionError, match="bf16 or f16"):
        backend.write_kv_cache(0, rows(1, KH).float(), rows(1, KH).float(), torch.zeros(1, dtype=torch.int64, device=DEV))
    pool.reset()
    assert all((s == 0).all() for s in pool.kv_scales)


def test_prefill_nan_values_reach_only_the_rows_that_attend_them():
    """NaN at some positions and columns of the values: NaN where a row attends them, nothing elsewhere."""
    H, KH, D, bs, c, n = 14, 2, 64, 16, 40, 300
    q, kc, vc, sc, table = prefill_case(6, [c], [n], (H, KH, D), bs, torch.bfloat16)
    at = [(130, 0, 3), (131, 0, 63), (250, 1, 17), (339, 1, 0)]  # position, KV head, column
    for p, h, d in at:
        bits(vc)[table[0, p // bs], h, p % bs, d] = 0xFF
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], [c], [n], bs)
    want = torch.zeros(n, H, D, dtype=torch.bool, device=DEV)
    for p, h, d in at:
        want[max(0, p - c):, h * 7:(h + 1) * 7, d] = True
        bits(vc)[table[0, p // bs], h, p % bs, d] = 0
    assert torch.equal(torch.isnan(out), want)
    k, v = F.dequant(kc, sc, 0, table[0], c + n), F.dequant(vc, sc, 1, table[0], c + n)
    ref, tol = F.attend(q, k, v, c + 1, D ** -0.5)
    F.check(torch.where(want, ref.to(q.dtype), out), ref, tol)


def test_prefill_value_scales_that_grow():
    """Value scales that rise by 2^9 from block to block, so that the accumulators' reference moves again and again."""
    H, KH, D, bs, n = 8, 2, 128, 16, 700
    q, kc, vc, sc, table = prefill_case(7, [0], [n], (H, KH, D), bs, torch.bfloat16)
    for i in range(44):
        sc[table[0, i], :, 1] *= 2.0 ** (-60 + 9 * (i // 8))
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], [0], [n], bs)
    # rows of the first 128 positions attend small values only, and are not lost beside what comes later
    check_prefill(out, q, kc, vc, sc, table, [0], [n], bs)


@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
def test_value_scales_that_jump_about(heads):
    """Value scales far apart in both directions, zeros (a block never written, a block of zeros) and small ones that
    count: decode, and prefill of the same queries."""
    lens = [700, 90]
    q, kc, vc, sc, table, kvl = decode_case(31, lens, heads, 16, torch.bfloat16)
    r = np.random.RandomState(5)
    for i, n in enumerate(lens):
        for b in range(-(-n // 16)):
            sc[table[i, b], :, 1] *= 2.0 ** float(r.randint(-14, 15))
    sc[table[0, 0], :, 1] = 0.0        # the first tile gives no reference
    sc[table[1, 0], :, 1] = 2.0 ** -100
    bits(vc)[table[1, 0]] = 0
    check_decode(M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16), q, kc, vc, sc, table, lens, 16)
    one = torch.ones(2, dtype=torch.int64, device=DEV)
    out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, one.cumsum(0) - 1, kvl.long() - 1, one, 16)
    check_decode(out, q, kc, vc, sc, table, lens, 16)


def test_decode_one_head_of_nan_leaves_the_others():
    lens = [600]
    q, kc, vc, sc, table, kvl = decode_case(32, lens, (14, 2, 64), 16, torch.bfloat16)
    sc[table[0, 20], :, 1] *= 2.0 ** 12
    q[0, 3] = math.nan
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    assert torch.isnan(out[0, 3]).all()
    keep = [h for h in range(14) if h != 3]
    k, v = (F.dequant(c, sc, w, table[0, :38], 600) for w, c in enumerate((kc, vc)))
    q[0, 3] = 0
    ref, tol = F.attend(q, k, v, 600, 0.125)
    F.check(out[:, keep], ref[:, keep], tol[:, keep])


# ---------------------------------------------------------------------------
# prefill of few rows: CTAs share a row tile's keys
# ---------------------------------------------------------------------------
FEW = {"one row": ([5000], [1]), "ragged": ([3000, 0, 255, 1000], [3, 1, 1, 20]), "no short share": ([4095], [1]),
       "empty shares": ([10, 5000], [3, 1]), "rows end in other shares": ([200], [300]),
       "with empty": ([2000, 70, 300], [9, 0, 30])}


@pytest.mark.parametrize("chunks", list(FEW))
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (16, 1, 128), (5, 5, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_of_few_rows(chunks, heads, dtype):
    cached, query = FEW[chunks]
    q, kc, vc, sc, table = prefill_case(40, cached, query, heads, 16, dtype, spare=2)
    n, rows = len(cached), sum(query)
    table = torch.cat([table, torch.full((n, 400), -1, dtype=table.dtype, device=DEV)], 1)  # wider than any needs
    size = _workspace_bytes(n, rows + 2, heads, 16, table.shape[1])
    assert size >= 2 * (rows + 2) * heads[0] * (heads[2] + 1) * 4  # two shares or more
    out = torch.full_like(q, 5.0)
    M.paged_prefill_attention_fp8(q, kc, vc, sc, table, list(range(n)), cached, query, 16, out=out)
    check_prefill(out[:rows], q, kc, vc, sc, table, cached, query, 16)
    assert (out[rows:] == 5.0).all()


def _workspace_bytes(chunks, total_q, heads, bs, max_blocks):
    size = ctypes.c_int64()
    assert _native.lib().mvb_paged_prefill_fp8_workspace(chunks, total_q, *heads, bs, max_blocks,
                                                         ctypes.byref(size)) == _native.OK
    return size.value


@pytest.mark.parametrize("bs", [128, 1024])
def test_prefill_of_few_rows_with_wide_scales(bs):
    """Scales that differ from share to share, and a query that makes one key win."""
    cached, query, heads = [2900], [40], (14, 2, 64)
    q, kc, vc, sc, table = prefill_case(41, cached, query, heads, bs, torch.bfloat16)
    sc *= torch.exp2(torch.randint(-6, 6, sc.shape, generator=gen(42), device=DEV).float())
    assert _workspace_bytes(1, 40, heads, bs, table.shape[1]) > 0
    for scale in (0.125, 2.0, -0.3):
        out = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], cached, query, bs, scale=scale)
        check_prefill(out, q, kc, vc, sc, table, cached, query, bs, scale=scale)


def test_prefill_of_few_rows_nan_and_errors():
    cached, query, (H, KH, D), bs = [1000], [30], (14, 2, 64), 16
    q, kc, vc, sc, table = prefill_case(43, cached, query, (H, KH, D), bs, torch.float16)
    assert _workspace_bytes(1, 30, (H, KH, D), bs, table.shape[1]) > 0
    call = lambda t, c=cached, n=query, **kw: M.paged_prefill_attention_fp8(q, kc, vc, sc, t, [0], c, n, bs, **kw)  # noqa: E731
    plain = call(table)
    for p, h, d in ((300, 0, 3), (1015, 1, 17)):  # in the first shares, and in the last one from row 15 on
        bits(vc)[table[0, p // bs], h, p % bs, d] = 0xFF
    out = call(table)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[:, :7, 3] = True
    want[15:, 7:, 17] = True
    assert torch.equal(torch.isnan(out), want)
    assert torch.equal(torch.where(want, 0, out), torch.where(want, 0, plain))
    q[4, 2, 5] = float("nan")
    out = call(table)
    want[4, 2] = True
    assert torch.equal(torch.isnan(out), want)
    with pytest.raises(IndexError, match="insufficient"):
        call(table, [1011], [30])  # 1041 positions, a table of 65 blocks
    out = call(table, [1100], [30], strict=False)
    assert (out == 0).all()
    with pytest.raises(IndexError):
        M.check_device_errors(DEV)
    out = torch.full_like(q, 5.0)
    with pytest.raises(IndexError):
        call(table, [900], [31], out=out)  # more tokens than query has rows
    assert (out == 5.0).all()
    t = table.clone()
    t[0, 10] = -1
    with pytest.raises(IndexError, match="block_table entry"):
        call(t)
    M.check_device_errors(DEV)


def test_prefill_of_few_rows_captured_on_two_streams():
    """Each call has results of its own between its kernels: two graphs at once, with an eager call between."""
    cases = [prefill_case(s, [3000, 500], [20, 7], (14, 2, 64), 16, torch.bfloat16) for s in (44, 45)]
    idx = [torch.tensor(x, device=DEV) for x in ([0, 1], [3000, 500], [20, 7])]
    want = [M.paged_prefill_attention_fp8(*c, *idx, 16) for c in cases]
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(M.paged_prefill_attention_fp8(*c, *idx, 16, strict=False))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = M.paged_prefill_attention_fp8(*cases[0], *idx, 16, strict=False)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(eager, want[0])


@pytest.mark.parametrize("lens,width", [([1000], 0), ([2048], 0), ([1, 16, 17, 700, 1000, 33], 0), ([0, 900, 0], 0),
                                        ([100] * 74, 0), ([100] * 75, 0), ([300, 40], 200), ([1, 5], 0)])
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 2, 64), (16, 2, 128), (24, 2, 128)])
def test_decode_of_few_short_sequences(lens, width, heads):
    """Units that a CTA takes whole, and lengths and tables beside the limits of that."""
    q, kc, vc, sc, table, kvl = decode_case(50, lens, heads, 16, torch.bfloat16)
    if width:
        table = torch.cat([table, torch.full((len(lens), width), -1, dtype=table.dtype, device=DEV)], 1)
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16, strict=False)
    kept = [i for i, n in enumerate(lens) if n > 0]
    check_decode(out[kept], q[kept], kc, vc, sc, table[kept], [lens[i] for i in kept], 16)
    assert all((out[i] == 0).all() for i, n in enumerate(lens) if n == 0)
    again = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16, strict=False)
    assert torch.equal(out, again)
    if 0 in lens:
        with pytest.raises(ValueError):
            M.check_device_errors(DEV)
    M.check_device_errors(DEV)


def test_scales_of_zero_and_lengths_past_any_table():
    """A block whose scale is 0 holds zeros; lengths near the integers' ends are refused, not followed."""
    lens, heads = [200, 90], (14, 2, 64)
    q, kc, vc, sc, table, kvl = decode_case(51, lens, heads, 16, torch.bfloat16)
    sc[table[0, 3]] = 0.0
    sc[table[0, 0], :, 1] = 0.0
    out = M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    check_decode(out, q, kc, vc, sc, table, lens, 16)
    rows, cached, one = (torch.tensor(x, device=DEV) for x in ([0, 1], [199, 89], [1, 1]))
    got = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, rows, cached, one, 16)
    check_prefill(got, q, kc, vc, sc, table, [199, 89], [1, 1], 16)
    for far in (2 ** 31 - 1, 2 ** 62, 2 ** 63 - 1):
        cached[0] = far
        with pytest.raises(IndexError):
            M.paged_prefill_attention_fp8(q, kc, vc, sc, table, rows, cached, one, 16)
    kvl[0] = 2 ** 31 - 1
    with pytest.raises(IndexError):
        M.paged_decode_attention_fp8(q, kc, vc, sc, table, kvl, 16)
    M.check_device_errors(DEV)


@pytest.mark.parametrize("n", [3, 100])
def test_captured_step_writes_then_attends(n):
    """A decode step in one graph (rotation and write, then attention), replayed as the sequences grow, against
    the same calls made one by one; the sequences share their first block."""
    H, KH, D, bs, width = 14, 2, 64, 16, 20
    g = gen(60)
    start = torch.randint(16, 290, (n,), generator=g, device=DEV)
    table = 1 + torch.arange(n * width, device=DEV).reshape(n, width)
    table[:, 0] = 0
    a = make_cache(g, n * width + 1, KH, bs, D)
    b = tuple(x.clone() for x in a)
    cos, sin = M.rope_tables(D, 10000.0, 512, torch.float32, DEV)
    rows = lambda h: torch.randn(n, h, D, generator=g, device=DEV).bfloat16()  # noqa: E731
    q, k, v, pos, slots = rows(H), rows(KH), rows(KH), start.clone(), torch.zeros_like(start)
    kvl = torch.zeros(n, dtype=torch.int32, device=DEV)

    def step(q, k, v, cache):
        qr, _ = M.rope_cache_write_fp8(q, k, v, pos, cos, sin, *cache, slots, bs, strict=False)
        return M.paged_decode_attention_fp8(qr, *cache, table, kvl, bs, strict=False)

    def at(p):  # the step of position p
        pos.copy_(p)
        slots.copy_(table.gather(1, (p // bs)[:, None])[:, 0] * bs + p % bs)
        kvl.copy_(p + 1)

    at(start)
    step(q, k, v, b)
    b = tuple(x.clone() for x in a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, k, v, a)
    for i in range(20):
        at(start + i)
        for x, h in ((q, H), (k, KH), (v, KH)):
            x.copy_(rows(h))
        graph.replay()
        want = step(q, k, v, b)
        assert torch.equal(out, want) and all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))
    check_decode(out, M.rope_cache_write_fp8(q, k, v, pos, cos, sin, *b, torch.full_like(slots, -1), bs)[0], *a, table,
                 kvl.tolist(), bs)
    M.check_device_errors(DEV)


def test_prefill_chunks_of_one_sequence():
    """The same row of the table twice, in any order of its chunks."""
    q, kc, vc, sc, table = prefill_case(61, [400], [100], (14, 2, 64), 16, torch.bfloat16)
    whole = M.paged_prefill_attention_fp8(q, kc, vc, sc, table, [0], [400], [100], 16)
    parts = torch.cat([q[60:], q[:60]])
    out = M.paged_prefill_attention_fp8(parts, kc, vc, sc, table, [0, 0], [460, 400], [40, 60], 16)
    check_prefill(out[:40], parts[:40], kc, vc, sc, table, [460], [40], 16)
    check_prefill(out[40:], parts[40:], kc, vc, sc, table, [400], [60], 16)
    check_prefill(whole, q, kc, vc, sc, table, [400], [100], 16)


@pytest.mark.parametrize("tokens", [1500, 4000])
def test_write_codes_are_those_of_the_exact_rotation(tokens):
    """Float32 tables: every key's code is that of the exact rotation rounded to float32, ties among 4 million too
    (a rotation by a rounded product and a fused multiply-add has another code about once in 2^20); infinities
    and NaN as ever."""
    g = gen(70)
    H, KH, D, bs = 8, 8, 128, 16
    kc, vc, sc = make_cache(g, tokens // bs + 1, KH, bs, D)
    mk, mv, ms = kc.cpu(), vc.cpu(), sc.cpu()
    q, k, v, pos, cos, sin = write_case(g, tokens, (H, KH, D), torch.bfloat16, torch.float32)
    slots = torch.arange(tokens, device=DEV)
    M.rope_cache_write_fp8(q, k, v, pos, cos, sin, kc, vc, sc, slots, bs)
    F.write(F.rotate(k, cos, sin, pos).cpu(), v.float().cpu(), mk, mv, ms, slots.cpu(), bs)
    for a, b in ((kc, mk), (vc, mv), (sc, ms)):
        assert torch.equal(bits(a).cpu(), bits(b))
    k = k.clone()
    k[3, 0, 5], k[4, 1, 70], pos[3:5] = float("inf"), float("nan"), 0  # (position 0: by cos 1 and sin 0)
    M.rope_cache_write_fp8(q, k, v, pos, cos, sin, kc, vc, sc, slots, bs)
    codes = kc[0].float()
    assert codes[0, 3, 5] == 448 and torch.isnan(codes[1, 4, 70]) and torch.isnan(codes[0]).sum() <= 1
