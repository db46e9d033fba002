"""The attention path over a KV cache held in 8 bits.

Half the bytes of a bf16 pool: twice the tokens in the same memory.  A decode takes
0.56 of the 16-bit one's time (with its per-step schedule, both in a graph) where reading
the cache is all of it (256 sequences of 32/8 heads of 128: 141 against 252 us), 0.65 for
32 sequences of 32768 tokens (59 against 91 us), 0.72 for one of 1000, but 0.87 for 256
sequences of up to 2048 (28.8 against 33.1 us), where half of it is set-up and merges.
The reference has no counterpart (its pool is 16 or 32 bits wide); names, arguments and
errors follow ``paged_attention_b200.py``.

The cache of one layer is three tensors:

* ``key_cache``, ``value_cache``: ``torch.float8_e4m3fn``
  ``[num_blocks, num_kv_heads, block_size, head_dim]``;
* ``kv_scale``: float32 ``[num_blocks, num_kv_heads, 2]``, the scale of the keys and
  of the values of each block and KV head.  An element stands for code * scale.

``KVCachePool.allocate(..., dtype=torch.float8_e4m3fn)`` makes all three, and
``AttentionBackendB200`` on such a pool calls the functions here.  They need
``head_dim`` 64 or 128, bf16 or f16 queries, keys and values, and a ``block_size``
that is a power of two from 16 to 1024.

Scales belong to whole blocks: ``paged_cache_write_fp8`` says how they follow the rows
that come in.  The writes make powers of two; the attention takes any positive normal
float32 scales, such as a calibration's (a block whose scale is 0 holds zeros).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .. import _native
from .paged_attention_b200 import (_DTYPE_CODES, _host_status, _raise_flags, _require, _state, _stream_handle,
                                   _take_flags)

FP8_DTYPE = torch.float8_e4m3fn
MIN_BLOCK_SIZE, MAX_BLOCK_SIZE = 16, 1024
_HALF = (torch.bfloat16, torch.float16)


def _check_cache(key_cache, value_cache, kv_scale, block_size, device) -> None:
    _require(key_cache.dim() == 4 and key_cache.shape == value_cache.shape,
             lambda: f"key_cache {tuple(key_cache.shape)} / value_cache {tuple(value_cache.shape)} mismatch")
    _require(key_cache.dtype == FP8_DTYPE and value_cache.dtype == FP8_DTYPE,
             lambda: f"caches must be float8_e4m3fn, got {key_cache.dtype} / {value_cache.dtype}")
    _require(key_cache.is_contiguous() and value_cache.is_contiguous(), "caches must be contiguous")
    num_blocks, num_kv_heads, bs, head_dim = key_cache.shape
    _require(head_dim in (64, 128), lambda: f"head_dim {head_dim} not supported (only 64, 128)")
    _require(MIN_BLOCK_SIZE <= block_size <= MAX_BLOCK_SIZE and (block_size & (block_size - 1)) == 0,
             lambda: f"block_size {block_size} must be a power of 2 from {MIN_BLOCK_SIZE} to {MAX_BLOCK_SIZE}")
    _require(bs == block_size, lambda: f"block_size {block_size} != cache dim2 {bs}")
    _require(num_blocks > 0 and num_kv_heads > 0, "the cache is empty")
    _require(kv_scale.shape == (num_blocks, num_kv_heads, 2) and kv_scale.dtype == torch.float32
             and kv_scale.is_contiguous(),
             lambda: f"kv_scale must be contiguous float32 [{num_blocks}, {num_kv_heads}, 2], got {kv_scale.dtype} "
                     f"{tuple(kv_scale.shape)}")
    _require(device.type == "cuda", lambda: f"tensors must be on a CUDA device, got {device}")
    _require(all(t.device == device for t in (key_cache, value_cache, kv_scale)),
             "caches, kv_scale and rows must be on one device")
    _require(key_cache.data_ptr() % 16 == 0 and value_cache.data_ptr() % 16 == 0 and kv_scale.data_ptr() % 8 == 0,
             "caches must be 16-byte and kv_scale 8-byte aligned")


def _aligned(x: torch.Tensor) -> bool:
    """Rows of 16-bit elements that the kernels read and write as 16-byte vectors."""
    return x.stride(2) == 1 and x.data_ptr() % 16 == 0 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if _aligned(x) else x.clone(memory_format=torch.contiguous_format)


def _int64(x: torch.Tensor, device) -> torch.Tensor:
    return x.to(device=device, dtype=torch.int64).contiguous()


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    """Scratch of one call, from the caching allocator on the current stream; it needs no initialisation."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _output(out: Optional[torch.Tensor], like: torch.Tensor, name: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """(tensor to return, tensor the kernel writes): the second is a copy where the rows are not aligned, which the
    caller copies back whole: rows that the kernel leaves alone keep what they held."""
    if out is None:
        out = torch.empty(like.shape, dtype=like.dtype, device=like.device)
        return out, out
    _require(out.shape == like.shape and out.dtype == like.dtype and out.device == like.device,
             lambda: f"{name} must match query's shape, dtype and device")
    _require(out.stride(2) == 1, lambda: f"{name}'s last dimension must be contiguous")
    return out, _rows(out)


def _raise_write(state, slot_mapping, key_cache, block_size, table_rows=None) -> None:
    flags = _take_flags(state)
    if flags:
        _raise_flags(flags, {"slot_mapping": slot_mapping, "total_slots": key_cache.shape[0] * block_size,
                             "block_size": block_size, "num_blocks": key_cache.shape[0], "table_rows": table_rows})


def _raise_read(state, max_blocks, key_cache, block_size, kv_len=None) -> None:
    flags = _take_flags(state)
    if flags:
        _raise_flags(flags, {"kv_len_after": kv_len, "max_blocks": max_blocks, "block_size": block_size,
                             "num_blocks": key_cache.shape[0]})


# ---------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------
def _check_write(key, value, key_cache, value_cache, kv_scale, slot_mapping, block_size) -> None:
    _require(key.dim() == 3 and key.shape == value.shape,
             lambda: f"key {tuple(key.shape)} / value {tuple(value.shape)} must be [num_tokens, num_kv_heads, head_dim]")
    _require(key.dtype in _HALF and value.dtype == key.dtype,
             lambda: f"key and value must both be bf16 or f16, got {key.dtype} / {value.dtype}")
    _require(value.device == key.device, "key and value must be on one device")
    _check_cache(key_cache, value_cache, kv_scale, block_size, key.device)
    _require(key.shape[1] == key_cache.shape[1] and key.shape[2] == key_cache.shape[3],
             lambda: f"key {tuple(key.shape)} does not match the cache {tuple(key_cache.shape)}")
    _require(slot_mapping.dim() == 1 and slot_mapping.shape[0] == key.shape[0],
             lambda: f"slot_mapping {tuple(slot_mapping.shape)} != ({key.shape[0]},)")


def _write_workspace(num_tokens: int, key_cache: torch.Tensor, block_size: int) -> Optional[torch.Tensor]:
    n = ctypes.c_int64()
    _host_status(_native.lib().mvb_kv_cache_write_fp8_workspace(num_tokens, key_cache.shape[0], block_size,
                                                                ctypes.byref(n)), "fp8 kv cache write")
    return _workspace(n.value, key_cache.device)


def paged_cache_write_fp8(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scale: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
    *,
    strict: bool = True,
) -> None:
    """Write per-token K/V rows into one layer's 8-bit cache, in place (``mvb_kv_cache_write_fp8``).

    Slots are those of ``paged_cache_write``.  For every block the call writes to, each KV head, and
    keys and values apart:

    * the scale becomes ``s``, the larger of the block's scale and the smallest power of two with which
      the largest of the call's (finite) elements fits 448; a call that writes slot 0 of a block starts
      it anew, whatever its scale was;
    * the new rows become ``round(x / s)``, to the nearest e4m3 value (an infinity becomes +-448 s);
    * where the scale has grown, the block's other rows are rounded anew: ``round(code * old / s)``.  That
      is exact but for values below ``2**-6 s``.

    So a block is filled from its slot 0 on, over any number of calls.  Two tokens with one slot raise
    ``AssertionError``, a slot outside the cache ``IndexError`` (with ``strict=False``: at
    ``check_device_errors``).  The call may be captured in a graph.  More than 2048 tokens take 4 bytes of
    scratch per slot of the cache from torch's allocator (a captured graph keeps its own), which
    ``compute_num_gpu_blocks`` leaves room for once.
    """
    fast = _native.fast()
    if fast is not None and key.is_cuda:
        state = _state(key.get_device())
        if fast.write_fp8(None, key, value, None, None, None, key_cache, value_cache, kv_scale, slot_mapping,
                          block_size, None, False, state.err_ptr)[0] == _native.OK:
            if strict:
                _raise_write(state, slot_mapping, key_cache, block_size)
            return
    _check_write(key, value, key_cache, value_cache, kv_scale, slot_mapping, block_size)
    if key.shape[0] == 0:
        return
    with torch.cuda.device(key.device):
        key, value, slot_mapping = _rows(key), _rows(value), _int64(slot_mapping, key.device)
        state = _state(key.get_device())
        ws = _write_workspace(key.shape[0], key_cache, block_size)
        status = _native.lib().mvb_kv_cache_write_fp8(
            key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
            key_cache.data_ptr(), value_cache.data_ptr(), kv_scale.data_ptr(), slot_mapping.data_ptr(), key.shape[0],
            key.shape[1], key.shape[2], block_size, key_cache.shape[0], _DTYPE_CODES[key.dtype],
            ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, state.err_ptr,
            _stream_handle(key.get_device()))
        _host_status(status, "fp8 kv cache write")
    if strict:
        _raise_write(state, slot_mapping, key_cache, block_size)


def rope_cache_write_fp8(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scale: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
    *,
    query_out: Optional[torch.Tensor] = None,
    return_key: bool = False,
    strict: bool = True,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RoPE of the step's query and key rows fused with ``paged_cache_write_fp8`` of the rotated keys and
    the values (``mvb_rope_kv_cache_write_fp8``).

    ``cos`` / ``sin`` are tables ``[rows, head_dim]`` (see ``rope_tables``) in the rows' dtype or in float32.
    The written keys' scales and codes are those of the exact rotation rounded to float32; the query and the
    returned keys are computed in float32 (a product and a fused multiply-add) and rounded to the rows' dtype
    (``rope_cache_write`` rounds after each operation, as the reference does).  Returns the rotated query (into
    ``query_out`` when given, which may be ``query`` itself and overlaps no other argument) and, with
    ``return_key``, the rotated keys.  A position outside the tables raises ``IndexError`` and leaves that token's
    rows unwritten; a token with slot -1 has its query rotated and writes nothing.
    """
    fast = _native.fast()
    if fast is not None and key.is_cuda:
        state = _state(key.get_device())
        status, q, k = fast.write_fp8(query, key, value, positions, cos, sin, key_cache, value_cache, kv_scale,
                                      slot_mapping, block_size, query_out, return_key, state.err_ptr)
        if status == _native.OK:
            if strict:
                _raise_write(state, slot_mapping, key_cache, block_size, cos.shape[0])
            return q, k
    _check_write(key, value, key_cache, value_cache, kv_scale, slot_mapping, block_size)
    num_tokens, num_kv_heads, head_dim = key.shape
    _require(query.dim() == 3 and query.shape[0] == num_tokens and query.shape[2] == head_dim and query.shape[1] > 0,
             lambda: f"query {tuple(query.shape)} does not match key {tuple(key.shape)}")
    _require(query.dtype == key.dtype and query.device == key.device, "query and key must share dtype and device")
    _require(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == head_dim and cos.shape[0] > 0,
             lambda: f"cos/sin tables {tuple(cos.shape)} / {tuple(sin.shape)} must be [rows, {head_dim}]")
    _require(cos.dtype == sin.dtype and cos.dtype in (key.dtype, torch.float32),
             lambda: f"cos/sin tables must be {key.dtype} or float32, got {cos.dtype} / {sin.dtype}")
    _require(cos.device == key.device and sin.device == key.device, "tables must be on the rows' device")
    _require(positions.dim() == 1 and positions.shape[0] == num_tokens,
             lambda: f"positions {tuple(positions.shape)} != ({num_tokens},)")
    with torch.cuda.device(key.device):
        out, target = _output(query_out, query, "query_out")
        key_out = torch.empty(key.shape, dtype=key.dtype, device=key.device) if return_key else None
        if num_tokens == 0:
            return out, key_out
        query, key, value = _rows(query), _rows(key), _rows(value)
        cos, sin = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                    for t in (cos, sin))
        positions, slot_mapping = _int64(positions, key.device), _int64(slot_mapping, key.device)
        state = _state(key.get_device())
        ws = _write_workspace(num_tokens, key_cache, block_size)
        status = _native.lib().mvb_rope_kv_cache_write_fp8(
            query.data_ptr(), query.stride(0), query.stride(1), target.data_ptr(), target.stride(0), target.stride(1),
            key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
            positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], _DTYPE_CODES[cos.dtype],
            key_cache.data_ptr(), value_cache.data_ptr(), kv_scale.data_ptr(), slot_mapping.data_ptr(),
            key_out.data_ptr() if key_out is not None else None, num_tokens, query.shape[1], num_kv_heads, head_dim,
            block_size, key_cache.shape[0], _DTYPE_CODES[key.dtype], ws.data_ptr() if ws is not None else None,
            ws.numel() if ws is not None else 0, state.err_ptr, _stream_handle(key.get_device()))
        _host_status(status, "rope + fp8 kv cache write")
        if target is not out:
            out.copy_(target)
    if strict:
        _raise_write(state, slot_mapping, key_cache, block_size, cos.shape[0])
    return out, key_out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _check_query(query, key_cache, value_cache, kv_scale, block_table, block_size, what) -> None:
    _require(query.dim() == 3, lambda: f"query must be [{what}, num_heads, head_dim], got {tuple(query.shape)}")
    _require(query.dtype in _HALF, lambda: f"query must be bf16 or f16, got {query.dtype}")
    _check_cache(key_cache, value_cache, kv_scale, block_size, query.device)
    _require(key_cache.shape[3] == query.shape[2],
             lambda: f"cache head_dim {key_cache.shape[3]} != query head_dim {query.shape[2]}")
    _require(query.shape[1] > 0 and query.shape[1] % key_cache.shape[1] == 0,
             lambda: f"num_q_heads {query.shape[1]} not divisible by num_kv_heads {key_cache.shape[1]}")
    _require(block_table.dim() == 2, lambda: f"block_table must be 2-D, got {tuple(block_table.shape)}")


def _table(block_table: torch.Tensor, device) -> torch.Tensor:
    block_table = block_table.to(device=device, dtype=torch.int64)
    return block_table if block_table.stride(1) == 1 and block_table.stride(0) >= block_table.shape[1] \
        else block_table.contiguous()


def paged_decode_attention_fp8(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scale: torch.Tensor,
    block_table: torch.Tensor,
    kv_len_after: torch.Tensor,
    block_size: int,
    scale: Optional[float] = None,
    *,
    out: Optional[torch.Tensor] = None,
    strict: bool = True,
) -> torch.Tensor:
    """Paged decode attention (one query token per sequence) over the 8-bit cache (``mvb_paged_decode_fp8``).

    Arguments, result and errors are ``paged_decode_attention``'s, with ``kv_scale`` beside the caches.  The
    query enters the tensor cores as f16 (a bf16 row by a power of two, exact but for elements below 2**-14 of
    its largest), probabilities as f16; logits, sums and the output are accumulated in float32.  Logits may be of any
    size in float32; those below its range count for nothing (a row with no others is zeros).  The result does not
    depend on timing.  At most 6144 sequences, and fewer than 2**31 cache rows (blocks * KV heads * block
    size).  The call keeps no state between calls and may be captured.
    """
    if scale is None:
        scale = query.shape[-1] ** -0.5
    fast = _native.fast()
    if fast is not None and query.is_cuda:
        state = _state(query.get_device())
        status, res = fast.decode_fp8(query, key_cache, value_cache, kv_scale, block_table, kv_len_after, block_size,
                                      float(scale), out, state.err_ptr)
        if status == _native.OK:
            if strict:
                _raise_read(state, block_table.shape[1], key_cache, block_size, kv_len_after)
            return res
    _check_query(query, key_cache, value_cache, kv_scale, block_table, block_size, "total_decode")
    n, num_heads, head_dim = query.shape
    _require(block_table.shape[0] == n, lambda: f"block_table rows {tuple(block_table.shape)} != total_decode {n}")
    _require(kv_len_after.shape == (n,), lambda: f"kv_len_after shape {tuple(kv_len_after.shape)} != ({n},)")
    dev = query.device
    with torch.cuda.device(dev):
        out, target = _output(out, query, "out")
        if n == 0:
            return out
        query, block_table = _rows(query), _table(block_table, dev)
        kv_len_after = kv_len_after.to(device=dev, dtype=torch.int32).contiguous()
        num_blocks, num_kv_heads = key_cache.shape[:2]
        shape = (n, num_heads, num_kv_heads, head_dim, block_size, num_blocks)
        nbytes = ctypes.c_int64()
        _host_status(_native.lib().mvb_paged_decode_fp8_workspace(
            *shape, block_table.shape[1], _DTYPE_CODES[query.dtype], ctypes.byref(nbytes)), "fp8 paged decode")
        ws = _workspace(nbytes.value, dev)
        state = _state(query.get_device())
        status = _native.lib().mvb_paged_decode_fp8(
            query.data_ptr(), query.stride(0), query.stride(1), key_cache.data_ptr(), value_cache.data_ptr(),
            kv_scale.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            kv_len_after.data_ptr(), target.data_ptr(), target.stride(0), target.stride(1), *shape, float(scale),
            _DTYPE_CODES[query.dtype], ws.data_ptr(), ws.numel(), state.err_ptr, _stream_handle(query.get_device()))
        _host_status(status, "fp8 paged decode")
        if target is not out:
            out.copy_(target)
    if strict:
        _raise_read(state, block_table.shape[1], key_cache, block_size, kv_len_after)
    return out


def paged_prefill_attention_fp8(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_rows,
    cached_len,
    query_len,
    block_size: int,
    *,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    strict: bool = True,
) -> torch.Tensor:
    """Causal prefill attention of a batch of chunks over the 8-bit cache (``mvb_paged_prefill_fp8``, no host
    synchronisation).

    Arguments and result are ``paged_prefill_attention``'s, with ``kv_scale`` beside the caches and without
    ``key`` / ``value``: every position is read from the cache, where the chunk has been written before.
    Token ``t`` of chunk ``i`` attends positions ``[0, cached_len[i] + t]``.  At most 4096 chunks; rows behind
    the last chunk's stay as they are.  Precision is ``paged_decode_attention_fp8``'s, but that a value whose
    block's scale is below ``2**-4`` of the sequence's largest keeps it as f16 in units of that one: exact down
    to ``2**-15`` of it.
    """
    _require(query.dim() == 3, lambda: f"query must be [total_q, num_heads, head_dim], got {tuple(query.shape)}")
    if scale is None:
        scale = query.shape[-1] ** -0.5
    fast = _native.fast()
    if fast is not None and query.is_cuda and all(isinstance(x, torch.Tensor) for x in (seq_rows, cached_len, query_len)):
        state = _state(query.get_device())
        status, res = fast.prefill_fp8(query, key_cache, value_cache, kv_scale, block_table, seq_rows, cached_len,
                                       query_len, block_size, float(scale), out, state.err_ptr)
        if status == _native.OK:
            if strict:
                _raise_read(state, block_table.shape[1], key_cache, block_size)
            return res
    _check_query(query, key_cache, value_cache, kv_scale, block_table, block_size, "total_q")
    dev = query.device
    with torch.cuda.device(dev):
        rows, cached, qlen = (_int64(x if isinstance(x, torch.Tensor) else torch.tensor(list(x), dtype=torch.int64), dev)
                              for x in (seq_rows, cached_len, query_len))
        n = rows.numel()
        _require(cached.numel() == n and qlen.numel() == n,
                 lambda: f"{n} sequences but {cached.numel()} cached lengths and {qlen.numel()} query lengths")
        out, target = _output(out, query, "out")
        total_q, num_heads, head_dim = query.shape
        if n == 0 or total_q == 0:
            return out
        query, block_table = _rows(query), _table(block_table, dev)
        num_blocks, num_kv_heads = key_cache.shape[:2]
        nbytes = ctypes.c_int64()
        _host_status(_native.lib().mvb_paged_prefill_fp8_workspace(
            n, total_q, num_heads, num_kv_heads, head_dim, block_size, block_table.shape[1], ctypes.byref(nbytes)),
            "fp8 paged prefill")
        ws = _workspace(nbytes.value, dev)
        state = _state(query.get_device())
        status = _native.lib().mvb_paged_prefill_fp8(
            query.data_ptr(), query.stride(0), query.stride(1), key_cache.data_ptr(), value_cache.data_ptr(),
            kv_scale.data_ptr(), block_table.data_ptr(), block_table.shape[0], block_table.stride(0),
            block_table.shape[1], rows.data_ptr(), cached.data_ptr(), qlen.data_ptr(), n, total_q, target.data_ptr(),
            target.stride(0), target.stride(1), num_heads, num_kv_heads, head_dim, block_size, num_blocks,
            float(scale), _DTYPE_CODES[query.dtype], ws.data_ptr() if ws is not None else 0, nbytes.value,
            state.err_ptr, _stream_handle(query.get_device()))
        _host_status(status, "fp8 paged prefill")
        if target is not out:
            out.copy_(target)
    if strict:
        _raise_read(state, block_table.shape[1], key_cache, block_size)
    return out
