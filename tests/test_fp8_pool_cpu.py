"""The 8-bit pool beside a model's settings (no GPU)."""

from __future__ import annotations

import pytest
import torch

import mini_vllm_b200 as M


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
def test_scales_are_float32_whatever_the_default(default):
    """A program that makes its model under another default dtype makes the pool under it too."""
    was = torch.get_default_dtype()
    try:
        torch.set_default_dtype(default)
        pool = M.KVCachePool.allocate(2, 16, 16, 2, 64, torch.float8_e4m3fn, torch.device("cpu"))
    finally:
        torch.set_default_dtype(was)
    assert all(s.dtype == torch.float32 for s in pool.kv_scales)


@pytest.mark.parametrize("layers,kv_heads", [(1, 1), (4, 2), (28, 2)])
def test_a_pool_that_fills_the_card_leaves_room_for_a_long_write(monkeypatch, layers, kv_heads):
    import ctypes

    from mini_vllm_b200 import _native

    free, reserve = 180 * 10 ** 9, 256 << 20
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda dev: (free, free))
    n = M.compute_num_gpu_blocks(layers, kv_heads, 64, 16, torch.float8_e4m3fn, torch.device("cuda"),
                                 gpu_memory_utilization=1.0, workspace_reserve=reserve)
    scratch = ctypes.c_int64()
    assert _native.lib().mvb_kv_cache_write_fp8_workspace(2049, n, 16, ctypes.byref(scratch)) == _native.OK
    pool = n * layers * kv_heads * (2 * 16 * 64 + 8)
    assert pool + scratch.value <= free - reserve
    assert pool + scratch.value > (free - reserve) * 0.999  # and no more than that
