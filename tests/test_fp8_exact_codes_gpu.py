"""Writes into the 8-bit cache compared bit for bit: every key's code is that of the exact rotation rounded to float32
(for 16-bit tables the products are exact in float32, for float32 tables the rounding errors are added back)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fp8_model as F
import mini_vllm_b200 as M
from test_fp8_cache_gpu import DEV, HEADS, bits, gen, make_cache, write_case

pytestmark = pytest.mark.gpu
TYPES = [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16)]


def check(heads, bs, types, slots, num_blocks, seed, calls=2):
    g = gen(seed)
    _, KH, D = heads
    kc, vc, sc = make_cache(g, num_blocks, KH, bs, D)
    mk, mv, ms = kc.cpu(), vc.cpu(), sc.cpu()
    slots = torch.as_tensor(slots, dtype=torch.int64, device=DEV)
    for _ in range(calls):
        q, k, v, pos, cos, sin = write_case(g, len(slots), heads, *types, rows=8192)
        M.rope_cache_write_fp8(q, k, v, pos, cos, sin, kc, vc, sc, slots, bs)
        F.write(F.rotate(k, cos, sin, pos).cpu(), v.float().cpu(), mk, mv, ms, slots.cpu(), bs)
        for a, b in ((kc, mk), (vc, mv), (sc, ms)):
            assert torch.equal(bits(a).cpu(), bits(b))


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("types", TYPES)
def test_ragged_chunks(heads, types):
    slots = list(range(5, 12)) + [16] + list(range(48, 64)) + [47, -1, 79]
    check(heads, 16, types, slots, 6, 1)


@pytest.mark.parametrize("bs", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("tokens", [1, 33, 300])
@pytest.mark.parametrize("types", TYPES)
def test_block_sizes_and_orders(bs, tokens, types):
    r = np.random.RandomState(bs + tokens)
    num_blocks = max(3, 2 * tokens // bs)
    slots = r.permutation(num_blocks * bs)[:tokens]
    slots[r.rand(tokens) < 0.1] = -1
    check((14, 2, 64), bs, types, slots, num_blocks, 2)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,tokens", [((14, 2, 64), 500), ((32, 8, 128), 500), ((14, 2, 64), 2200)])
def test_one_row_per_block(heads, tokens, types):
    r = np.random.RandomState(tokens)
    check(heads, 16, types, r.permutation(tokens) * 16 + r.randint(0, 16, tokens), tokens, 3)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,bs,tokens", [((14, 2, 64), 16, 6000), ((16, 8, 128), 64, 2500)])
def test_many_tokens(heads, bs, tokens, types):
    check(heads, bs, types, np.arange(3, tokens + 3), tokens // bs + 2, 4, calls=1)
