"""A paged key/value cache on the gfx950 HIP kernels ``fd_paged_kv_write`` and ``fd_paged_kv_read``.

The reference keeps the keys and values of a shared prefix in transformers' cache and
forks it per question (ref: src/decider/shared_prefix.py); here a cache is a pool of
pages that requests hold through a page table:

* ``k_cache``, ``v_cache`` — logical ``[n_pages, Hkv, page_size, D]`` (any strides with a
  contiguous feature dimension, the same for both), bf16 or ``torch.float8_e4m3fn``; D 64, 128 or 256,
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

import torch

from . import _cache_lib, _lib

HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)
_BF16, _E4M3, _INT32, _UINT8 = torch.bfloat16, torch.float8_e4m3fn, torch.int32, torch.uint8


def check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, requests) -> bytes:
    """Validate a cache and its page table for ``requests`` requests; the packed ``fd_paged_cache``."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must be [n_pages, Hkv, page_size, D] of one shape")
    n_pages, heads, page_size, dim = shape
    device = k_cache.get_device()
    if device < 0 or v_cache.get_device() != device:
        raise ValueError("The caches must share a CUDA device")
    dtype = k_cache.dtype
    if (dtype != _BF16 and dtype != _E4M3) or v_cache.dtype != dtype:
        raise ValueError("The caches must both be BF16 or float8_e4m3fn")
    if dim not in HEAD_DIMS:
        raise ValueError("The cache's head dimension must be 64, 128 or 256")
    if page_size not in PAGE_SIZES:
        raise ValueError("page_size must be a power of two in [16, 256]")
    if n_pages < 1 or heads < 1:
        raise ValueError("The cache needs at least one page and one head")
    fp8 = dtype == _E4M3
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    strides = k_cache.stride()
    if v_cache.stride() != strides:
        raise ValueError("k_cache and v_cache must have the same strides")
    sp, sh, sr, sd = strides
    if sd != 1 or (k_ptr | v_ptr) % 16 or (sp | sh | sr) % (16 if fp8 else 8) or sr >= 1 << 20:
        raise ValueError("Cache rows must be contiguous and 16-byte aligned")
    ks = vs = ssp = ssh = 0
    if fp8:
        for t in (k_scale, v_scale):
            if (t is None or t.shape != shape[:3] or t.dtype != _UINT8 or t.get_device() != device or t.stride(2) != 1):
                raise ValueError("An e4m3 cache needs k_scale and v_scale: uint8 [n_pages, Hkv, page_size] on its device")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
        if v_scale.stride() != k_scale.stride():
            raise ValueError("k_scale and v_scale must have the same strides")
        ssp, ssh, _ = k_scale.stride()
    elif k_scale is not None or v_scale is not None:
        raise ValueError("A BF16 cache has no scales")
    max_pages = page_table.shape[-1]
    table_stride = page_table.stride()
    if (page_table.shape != (requests, max_pages) or max_pages < 1 or page_table.dtype != _INT32
            or page_table.get_device() != device or table_stride[1] != 1):
        raise ValueError(f"page_table must be int32 [{requests}, max_pages] on the cache's device, its rows contiguous")
    if max_pages * page_size >= 1 << 27:
        raise ValueError("A request holds fewer than 2^27 keys")
    lens = 0
    if cache_lens is not None:
        if (cache_lens.shape != (requests,) or cache_lens.dtype != _INT32 or cache_lens.get_device() != device
                or not cache_lens.is_contiguous()):
            raise ValueError(f"cache_lens must be a contiguous int32 vector [{requests}] on the cache's device")
        lens = cache_lens.data_ptr()
    return _cache_lib.pack_cache(k_ptr, v_ptr, ks, vs, sp, sh, sr, sp, sh, sr, ssp, ssh, ssp, ssh, page_table.data_ptr(),
                                 table_stride[0], lens, n_pages, page_size, max_pages, heads, dim,
                                 _cache_lib.FD_DTYPE_E4M3 if fp8 else _lib.FD_DTYPE_BF16)


def check_cu_seqlens(cu_seqlens, batch, device) -> tuple[int | None, int]:
    """(pointer, n_seqs) of an offset vector on device ``device`` (an index); (None, 0) without one."""
    if cu_seqlens is None:
        return None, 0
    if batch != 1:
        raise ValueError("cu_seqlens requires batch size 1 (packed requests)")
    if (cu_seqlens.ndim != 1 or cu_seqlens.dtype != _INT32 or cu_seqlens.get_device() != device
            or cu_seqlens.numel() < 2 or not cu_seqlens.is_contiguous()):
        raise ValueError("cu_seqlens must be a contiguous int32 vector [n_seqs + 1] on the cache's device")
    return cu_seqlens.data_ptr(), cu_seqlens.numel() - 1


def check_rows(name: str, t: torch.Tensor, shape, device: int) -> tuple[int, bytes]:
    """(pointer, packed strides) of a bf16 tensor of rows."""
    if t.shape != shape or t.dtype != _BF16 or t.get_device() != device:
        raise ValueError(f"{name} must be BF16 {list(shape)} on the cache's device")
    strides, ptr = t.stride(), t.data_ptr()
    sb, sh, st, sd = strides
    if sd != 1 or ptr % 16 or (sb | sh | st) % 8:
        raise ValueError(f"{name} rows must be contiguous and 16-byte aligned")
    return ptr, _cache_lib.pack4(*strides)


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
    shape = key.shape
    if len(shape) != 4 or k_cache.ndim != 4 or value.shape != shape:
        raise ValueError("key and value must be [B, Hkv, T, D] of one shape")
    batch, heads, seq_len, dim = shape
    if batch < 1 or seq_len < 1:
        raise ValueError("Batch and sequence length must be positive")
    if heads != k_cache.shape[1] or dim != k_cache.shape[3]:
        raise ValueError("key and value must have the cache's heads and head dimension")
    if cache_lens is None:
        raise ValueError("cache_lens is required")
    device = k_cache.get_device()
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, batch, device)
    cache = check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, n_seqs or batch)
    k_ptr, k_strides = check_rows("key", key, shape, device)
    v_ptr, v_strides = check_rows("value", value, shape, device)
    if _cache_lib.current_device() != device:
        with torch.cuda.device(device):
            return paged_kv_write(key, value, k_cache, v_cache, page_table, cache_lens, k_scale=k_scale, v_scale=v_scale,
                                  cu_seqlens=cu_seqlens)
    _cache_lib.check("fd_paged_kv_write", _cache_lib.lib().fd_paged_kv_write(
        k_ptr, v_ptr, k_strides, v_strides, cache, batch, seq_len, cu_ptr, n_seqs, _cache_lib.raw_stream(device)))


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
    device = k_cache.get_device()
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, 1, device)
    if n_seqs == 0:
        raise ValueError("cu_seqlens is required")
    total = int(total)
    if not 0 <= total < 1 << 31:
        raise ValueError("total must be in [0, 2^31)")
    cache = check_cache(k_cache, v_cache, page_table, None, k_scale, v_scale, n_seqs)
    if _cache_lib.current_device() != device:
        with torch.cuda.device(device):
            return paged_kv_read(k_cache, v_cache, page_table, cu_seqlens, total, k_scale=k_scale, v_scale=v_scale)
    _, heads, _, dim = k_cache.shape
    strides = (total * heads * dim, dim, heads * dim, 1)
    k = torch.empty_strided((1, heads, total, dim), strides, device=k_cache.device, dtype=_BF16)
    v = torch.empty_like(k)
    if total == 0:
        return k, v
    at = _cache_lib.pack2(dim, heads * dim)
    _cache_lib.check("fd_paged_kv_read", _cache_lib.lib().fd_paged_kv_read(
        cache, k.data_ptr(), v.data_ptr(), at, at, total, cu_ptr, n_seqs, _cache_lib.raw_stream(device)))
    return k, v
