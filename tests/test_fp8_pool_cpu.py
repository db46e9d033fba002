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
