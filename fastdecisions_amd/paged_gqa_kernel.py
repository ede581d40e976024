"""Grouped-query attention of new tokens over a paged cache on the gfx950 HIP kernel ``fd_paged_gqa_fwd``.

What ``native_gqa_attention`` is to a whole prompt, ``paged_gqa_attention`` is to the
tokens that continue one (ref: src/decider/shared_prefix.py runs suffixes over a cached
prefix through transformers' attention): a single token, a suffix or the next piece of
a long prompt, causal over everything the request holds.  The new tokens' own keys and
values are in the cache already (``paged_kv_write`` with the same ``cache_lens``):

* q logical ``[B, Hq, T, D]`` bf16, any strides with contiguous rows; Hq a multiple of
  the cache's heads; the output is a ``[B, Hq, T, D]`` view of a physical ``[B, T, Hq, D]``;
* without ``cu_seqlens`` request r is batch row r with T new tokens; with it (B == 1) T
  packs the requests' new tokens, and ``max_seqlen`` (the longest request's, default T)
  says which kernel suits the call: it bounds nothing.  Output rows behind the last request
  are not written;
* new token i of n of request r sees the keys ``0 .. cache_lens[r] - n + i`` that lie on a
  page; a row that sees none is zeros;
* ``gate`` (logically like the output): ``attention * sigmoid(gate)``, rounded once.

The cache's layout is described in ``paged_kv_kernel``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _cache_lib, _lib
from .paged_kv_kernel import check_cache, check_cu_seqlens


def paged_gqa_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    *,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    scale: float | None = None,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
    gate: torch.Tensor | None = None,
) -> torch.Tensor:
    if q.ndim != 4:
        raise ValueError("Q must be four-dimensional")
    batch, q_heads, seq_len, dim = q.shape
    if min(batch, q_heads, seq_len) < 1:
        raise ValueError("Batch, head counts and sequence length must be positive")
    if k_cache.ndim != 4 or q_heads % k_cache.shape[1] or dim != k_cache.shape[3]:
        raise ValueError("Q must have the cache's head dimension and a multiple of its heads")
    for name, t in (("Q", q), ("gate", gate)):
        if t is None:
            continue
        if t.shape != q.shape or t.dtype != torch.bfloat16 or t.device != k_cache.device:
            raise ValueError(f"{name} must be BF16, shaped like Q, on the cache's device")
        sb, sh, st, sd = t.stride()
        if sd != 1 or t.data_ptr() % 16 or (sb | sh | st) % 8:
            raise ValueError(f"{name} rows must be contiguous and 16-byte aligned")
    if batch * seq_len * q_heads >= 1 << 30:
        raise ValueError("B * T * Hq must be below 2^30")
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, batch, k_cache.device)
    if max_seqlen is None or n_seqs == 0:
        max_seqlen = seq_len
    if not 0 <= int(max_seqlen) <= seq_len:
        raise ValueError("max_seqlen must lie in [0, T]")
    if scale is None:
        scale = dim ** -0.5
    if not 0.0 < scale < 1e30:
        raise ValueError("scale must be positive")
    if cache_lens is None:
        raise ValueError("cache_lens is required")
    cache = check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, n_seqs or batch)
    with _lib.on_device(q.device):
        out = torch.empty((batch, seq_len, q_heads, dim), device=q.device, dtype=q.dtype).permute(0, 2, 1, 3)
        lib = _cache_lib.lib()
        nbytes = lib.fd_paged_gqa_workspace_bytes(batch, q_heads, cache.kv_heads, seq_len, dim, cache.page_size,
                                                  cache.max_pages, n_seqs, int(max_seqlen))
        _cache_lib.check("fd_paged_gqa_workspace_bytes", nbytes)
        work = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes > 0 else None
        _cache_lib.check("fd_paged_gqa_fwd", lib.fd_paged_gqa_fwd(
            q.data_ptr(), ctypes.byref(cache), _lib.ptr(gate), out.data_ptr(), _lib.strides4(q),
            None if gate is None else _lib.strides4(gate), _lib.strides4(out), batch, q_heads, seq_len, float(scale),
            cu_ptr, n_seqs, int(max_seqlen), _lib.ptr(work), nbytes, _lib.stream_handle(q.device)))
    return out
