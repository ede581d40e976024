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

from functools import lru_cache

import torch

from . import _cache_lib
from .paged_kv_kernel import check_cache, check_cu_seqlens, check_rows


@lru_cache(maxsize=4096)
def workspace_bytes(batch: int, q_heads: int, kv_heads: int, seq_len: int, head_dim: int, page_size: int,
                    max_pages: int, n_seqs: int, max_seqlen: int) -> int:
    """Device workspace of a call of these sizes (``fd_paged_gqa_workspace_bytes``)."""
    nbytes = _cache_lib.lib().fd_paged_gqa_workspace_bytes(batch, q_heads, kv_heads, seq_len, head_dim, page_size,
                                                           max_pages, n_seqs, max_seqlen)
    _cache_lib.check("fd_paged_gqa_workspace_bytes", nbytes)
    return nbytes


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
    shape = q.shape
    if len(shape) != 4:
        raise ValueError("Q must be four-dimensional")
    batch, q_heads, seq_len, dim = shape
    if min(batch, q_heads, seq_len) < 1:
        raise ValueError("Batch, head counts and sequence length must be positive")
    if k_cache.ndim != 4:
        raise ValueError("k_cache and v_cache must be [n_pages, Hkv, page_size, D] of one shape")
    _, kv_heads, page_size, cache_dim = k_cache.shape
    if kv_heads < 1 or q_heads % kv_heads or dim != cache_dim:
        raise ValueError("Q must have the cache's head dimension and a multiple of its heads")
    if q_heads // kv_heads > 2048:
        raise ValueError("at most 2048 query heads per key head")
    if batch * seq_len * q_heads >= 1 << 30:
        raise ValueError("B * T * Hq must be below 2^30")
    if scale is None:
        scale = dim ** -0.5
    elif not 0.0 < scale < 1e30:
        raise ValueError("scale must be positive")
    if cache_lens is None:
        raise ValueError("cache_lens is required")
    device = k_cache.get_device()
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, batch, device)
    if max_seqlen is None or n_seqs == 0:
        max_seqlen = seq_len
    elif not 0 <= int(max_seqlen) <= seq_len:
        raise ValueError("max_seqlen must lie in [0, T]")
    cache = check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, n_seqs or batch)
    q_ptr, q_strides = check_rows("Q", q, shape, device)
    g_ptr, g_strides = (None, None) if gate is None else check_rows("gate", gate, shape, device)
    if _cache_lib.current_device() != device:
        with torch.cuda.device(device):
            return paged_gqa_attention(q, k_cache, v_cache, page_table, cache_lens, k_scale=k_scale, v_scale=v_scale,
                                       scale=scale, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, gate=gate)
    strides = (seq_len * q_heads * dim, dim, q_heads * dim, 1)
    out = torch.empty_strided(shape, strides, device=q.device, dtype=q.dtype)
    nbytes = workspace_bytes(batch, q_heads, kv_heads, seq_len, dim, page_size, page_table.shape[1], n_seqs,
                             int(max_seqlen))
    work = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes > 0 else None
    _cache_lib.check("fd_paged_gqa_fwd", _cache_lib.lib().fd_paged_gqa_fwd(
        q_ptr, cache, g_ptr, out.data_ptr(), q_strides, g_strides, _cache_lib.pack4(*strides), batch, q_heads, seq_len,
        float(scale), cu_ptr, n_seqs, int(max_seqlen), None if work is None else work.data_ptr(), nbytes,
        _cache_lib.raw_stream(device)))
    return out
