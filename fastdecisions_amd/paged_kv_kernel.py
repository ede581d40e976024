"""A paged key/value cache on the gfx950 HIP kernels ``fd_paged_kv_write`` and ``fd_paged_kv_read``.

The reference keeps the keys and values of a shared prefix in transformers' cache and
forks it per question (ref: src/decider/shared_prefix.py); here a cache is a pool of
pages that requests hold through a page table:

* ``k_cache``, ``v_cache`` — logical ``[n_pages, Hkv, page_size, D]`` (any strides with a
  contiguous feature dimension), bf16 or ``torch.float8_e4m3fn``; D 64, 128 or 256,
  page_size a power of two in [16, 256];
* ``k_scale``, ``v_scale`` — for an e4m3 cache, uint8 ``[n_pages, Hkv, page_size]``: byte b
  stands for 2^(b - 127), and a cached value is its code times that;
* ``page_table`` — int32 ``[requests, max_pages]``; key j of request r is row
  ``j % page_size`` of page ``page_table[r, j // page_size]``.  An entry outside
  ``[0, n_pages)`` (as -1) is no page: its keys are not written, read as zeros and are
  not visible to attention;
* ``cache_lens`` — int32 ``[requests]``: the keys each request holds, the new tokens of
  the call included.

``paged_kv_write(key, value, ...)`` writes the new tokens' keys and values (logical
``[B, Hkv, T, D]`` bf16, any strides with contiguous rows, as ``native_gqa_attention``
takes them) as the last keys of their requests; with ``cu_seqlens`` (B == 1) T packs the
requests' new tokens, else request r is batch row r.  ``paged_kv_read`` returns the first
keys and values of every request as dense bf16 tensors.  Two requests of one call must
not write the same rows of a shared page; they may read whatever they share.
"""
from __future__ import annotations

import ctypes

import torch

from . import _cache_lib, _lib

HEAD_DIMS = (64, 128, 256)


def check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, requests) -> _cache_lib.PagedCache:
    """Validate a cache and its page table for ``requests`` requests; the struct the library takes."""
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must be [n_pages, Hkv, page_size, D] of one shape")
    n_pages, heads, page_size, dim = k_cache.shape
    if not k_cache.is_cuda or v_cache.device != k_cache.device:
        raise ValueError("The caches must share a CUDA device")
    if k_cache.dtype not in (torch.bfloat16, torch.float8_e4m3fn) or v_cache.dtype != k_cache.dtype:
        raise ValueError("The caches must both be BF16 or float8_e4m3fn")
    if dim not in HEAD_DIMS:
        raise ValueError("The cache's head dimension must be 64, 128 or 256")
    if not 16 <= page_size <= 256 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two in [16, 256]")
    if n_pages < 1 or heads < 1:
        raise ValueError("The cache needs at least one page and one head")
    size = k_cache.element_size()
    for t in (k_cache, v_cache):
        sp, sh, sr, sd = t.stride()
        if sd != 1 or t.data_ptr() % 16 or (sp | sh | sr) * size % 16 or not 0 <= sr < 1 << 20:
            raise ValueError("Cache rows must be contiguous and 16-byte aligned")
    c = _cache_lib.PagedCache()
    c.dtype = _lib.FD_DTYPE_BF16
    if k_cache.dtype == torch.float8_e4m3fn:
        c.dtype = _cache_lib.FD_DTYPE_E4M3
        for t in (k_scale, v_scale):
            if (t is None or t.dtype != torch.uint8 or t.device != k_cache.device
                    or t.shape != (n_pages, heads, page_size) or t.stride(2) != 1):
                raise ValueError("An e4m3 cache needs k_scale and v_scale: uint8 [n_pages, Hkv, page_size] on its device")
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        c.k_scale_strides[:] = k_scale.stride()[:2]
        c.v_scale_strides[:] = v_scale.stride()[:2]
    elif k_scale is not None or v_scale is not None:
        raise ValueError("A BF16 cache has no scales")
    if (page_table.ndim != 2 or page_table.dtype != torch.int32 or page_table.device != k_cache.device
            or page_table.shape[0] != requests or page_table.shape[1] < 1 or page_table.stride(1) != 1):
        raise ValueError(f"page_table must be int32 [{requests}, max_pages] on the cache's device, its rows contiguous")
    if page_table.shape[1] * page_size >= 1 << 27:
        raise ValueError("A request holds fewer than 2^27 keys")
    if cache_lens is not None:
        if (cache_lens.shape != (requests,) or cache_lens.dtype != torch.int32 or cache_lens.device != k_cache.device
                or not cache_lens.is_contiguous()):
            raise ValueError(f"cache_lens must be a contiguous int32 vector [{requests}] on the cache's device")
        c.cache_lens = cache_lens.data_ptr()
    c.k, c.v = k_cache.data_ptr(), v_cache.data_ptr()
    c.k_strides[:] = k_cache.stride()[:3]
    c.v_strides[:] = v_cache.stride()[:3]
    c.page_table, c.table_stride = page_table.data_ptr(), page_table.stride(0)
    c.n_pages, c.kv_heads, c.page_size, c.head_dim = n_pages, heads, page_size, dim
    c.max_pages = page_table.shape[1]
    return c


def check_cu_seqlens(cu_seqlens, batch, device) -> tuple[int | None, int]:
    """(pointer, n_seqs) of an offset vector; (None, 0) without one."""
    if cu_seqlens is None:
        return None, 0
    if batch != 1:
        raise ValueError("cu_seqlens requires batch size 1 (packed requests)")
    if (cu_seqlens.ndim != 1 or cu_seqlens.dtype != torch.int32 or cu_seqlens.device != device
            or cu_seqlens.numel() < 2 or not cu_seqlens.is_contiguous()):
        raise ValueError("cu_seqlens must be a contiguous int32 vector [n_seqs + 1] on the cache's device")
    return cu_seqlens.data_ptr(), cu_seqlens.numel() - 1


def paged_kv_write(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    *,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
) -> None:
    if key.ndim != 4 or k_cache.ndim != 4 or value.shape != key.shape:
        raise ValueError("key and value must be [B, Hkv, T, D] of one shape")
    batch, heads, seq_len, dim = key.shape
    if heads != k_cache.shape[1] or dim != k_cache.shape[3]:
        raise ValueError("key and value must have the cache's heads and head dimension")
    for t in (key, value):
        if t.dtype != torch.bfloat16 or t.device != k_cache.device:
            raise ValueError("key and value must be BF16 on the cache's device")
        sb, sh, st, sd = t.stride()
        if sd != 1 or t.data_ptr() % 16 or (sb | sh | st) % 8:
            raise ValueError("key and value rows must be contiguous and 16-byte aligned")
    if cache_lens is None:
        raise ValueError("cache_lens is required")
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, batch, k_cache.device)
    cache = check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, n_seqs or batch)
    with _lib.on_device(k_cache.device):
        _cache_lib.check("fd_paged_kv_write", _cache_lib.lib().fd_paged_kv_write(
            key.data_ptr(), value.data_ptr(), _lib.strides4(key), _lib.strides4(value), ctypes.byref(cache), batch,
            seq_len, cu_ptr, n_seqs, _lib.stream_handle(k_cache.device)))


def paged_kv_read(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    total: int,
    *,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys 0 .. cu_seqlens[r + 1] - cu_seqlens[r] - 1 of every request r as rows ``cu_seqlens[r]`` ..
    of ``[1, Hkv, total, D]`` bf16 keys and values (physical ``[1, total, Hkv, D]``).  Keys on no page
    are zeros; rows from ``cu_seqlens[-1]`` on are not written."""
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, 1, k_cache.device)
    if n_seqs == 0:
        raise ValueError("cu_seqlens is required")
    if not 0 <= int(total) < 1 << 31:
        raise ValueError("total must be in [0, 2^31)")
    cache = check_cache(k_cache, v_cache, page_table, None, k_scale, v_scale, n_seqs)
    with _lib.on_device(k_cache.device):
        k, v = (torch.empty((1, int(total), cache.kv_heads, cache.head_dim), device=k_cache.device,
                            dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
        at = (ctypes.c_int64 * 2)(cache.head_dim, cache.kv_heads * cache.head_dim)
        _cache_lib.check("fd_paged_kv_read", _cache_lib.lib().fd_paged_kv_read(
            ctypes.byref(cache), k.data_ptr(), v.data_ptr(), at, at, int(total), cu_ptr, n_seqs,
            _lib.stream_handle(k_cache.device)))
    return k, v
