"""Which cached keys matter, and a cache without the others, on the gfx950 HIP kernels ``fd_paged_key_weights`` and
``fd_paged_kv_evict``.

``paged_key_weights`` adds to each cached key the attention weight that a call's new tokens give it:
the sum over the tokens and over the query heads of a key head of their softmax probabilities, in
fp32.  It takes what ``paged_gqa_attention`` takes, after ``paged_kv_write`` of the same tokens:

* ``weights`` — fp32 ``[rows, Hkv, width]``, keys contiguous, ``width`` at least
  ``max_pages * page_size``; key j of request r is ``weights[row_indices[r], h, j]`` (int32, default
  row r).  It belongs to a request, not to a page: requests that share pages weigh them apart.  An
  index outside the rows, or named by an earlier request of the call, adds nothing;
* ``last`` — only the last ``last`` new tokens of each request count (default: all).

``paged_kv_evict`` cuts every request to at most ``keep`` keys: its ``recent`` last ones and, per key
head, those of largest weight among the others (of equal weights the lowest; NaN below everything).
Their rows and scales move, in their order, to the pages of ``new_table`` (int32 ``[requests, n]``,
``n * page_size >= keep``), which must be distinct and none of those that hold the call's requests; the old
pages are left as they were.  A request without a row of weights counts as one of equal weights.  A request of no more than ``keep`` keys moves whole.  Keys are rotated by their
positions before they are cached, so a request goes on where it stood: its next tokens' positions count
all the tokens that it has seen, ``cache_lens`` those that it holds.

* returns ``(kept, new_lens)``: int32 ``[requests, Hkv, keep]``, the old place of every kept key (-1
  behind the last), and int32 ``[requests]``, ``min(cache_lens, keep)``;
* ``weights_out`` (default ``weights`` itself) — the kept keys' weights in the first places of their rows,
  zeros from there to ``cache_lens``.

The cache's layout is described in ``paged_kv_kernel``.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _cache_lib
from .paged_kv_kernel import cache_dim, check_cache, check_cu_seqlens, check_rows


@lru_cache(maxsize=4096)
def workspace_bytes(batch: int, q_heads: int, kv_heads: int, seq_len: int, head_dim: int, page_size: int, max_pages: int,
                    n_seqs: int, max_seqlen: int, last: int) -> int:
    """Device workspace of a call of these sizes (``fd_paged_key_weights_workspace_bytes``)."""
    nbytes = _cache_lib.lib().fd_paged_key_weights_workspace_bytes(batch, q_heads, kv_heads, seq_len, head_dim, page_size,
                                                                   max_pages, n_seqs, max_seqlen, last)
    _cache_lib.check("fd_paged_key_weights_workspace_bytes", nbytes)
    return nbytes


def check_weights(name, weights, heads, width, device) -> tuple[int, bytes]:
    """(rows, packed strides) of the weights."""
    shape, strides = weights.shape, weights.stride()
    if (len(shape) != 3 or weights.dtype is not torch.float32 or weights.get_device() != device or shape[1] != heads
            or shape[2] < width or strides[2] != 1):
        raise ValueError(f"{name} must be FP32 [rows, {heads}, at least {width}] on the cache's device, its keys contiguous")
    (row, head, _), (rows, _, keys) = strides, shape
    if (rows > 1 and row < keys) or (heads > 1 and head < keys) or (rows > 1 and heads > 1 and row < heads * head and head < rows * row):
        raise ValueError(f"{name} must not hold two of its elements in the same memory")
    return rows, _cache_lib.pack2(row, head)


def check_row_indices(row_indices, requests, rows, device) -> int | None:
    if row_indices is None:
        if rows < requests:
            raise ValueError(f"Without row_indices the weights need a row for each of the {requests} requests")
        return None
    if (row_indices.shape != (requests,) or row_indices.dtype != torch.int32 or row_indices.get_device() != device
            or not row_indices.is_contiguous()):
        raise ValueError(f"row_indices must be a contiguous int32 vector [{requests}] on the cache's device")
    return row_indices.data_ptr()


def paged_key_weights(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    weights: torch.Tensor,
    *,
    k_scale: torch.Tensor | None = None,
    scale: float | None = None,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
    last: int | None = None,
    row_indices: torch.Tensor | None = None,
) -> None:
    shape = q.shape
    if len(shape) != 4:
        raise ValueError("Q must be four-dimensional")
    batch, q_heads, seq_len, dim = shape
    if batch < 1 or q_heads < 1 or seq_len < 1:
        raise ValueError("Batch, head counts and sequence length must be positive")
    if k_cache.ndim != 4:
        raise ValueError("k_cache must be [n_pages, Hkv, page_size, D]")
    _, kv_heads, page_size, _ = k_cache.shape
    if kv_heads < 1 or q_heads % kv_heads or dim != cache_dim(k_cache):
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
    if last is not None and not 1 <= int(last) < 1 << 31:
        raise ValueError("last must be a positive number of tokens")
    device = k_cache.get_device()
    cu_ptr, n_seqs = check_cu_seqlens(cu_seqlens, batch, device)
    if max_seqlen is None or n_seqs == 0:
        max_seqlen = seq_len
    elif not 0 <= int(max_seqlen) <= seq_len:
        raise ValueError("max_seqlen must lie in [0, T]")
    requests = n_seqs or batch
    cache = check_cache(k_cache, k_cache, page_table, cache_lens, k_scale, k_scale, requests)
    max_pages = page_table.shape[1]
    rows, w_strides = check_weights("weights", weights, kv_heads, max_pages * page_size, device)
    index = check_row_indices(row_indices, requests, rows, device)
    q_ptr, q_strides = check_rows("Q", q, shape, device)
    if _cache_lib.current_device() != device:
        with torch.cuda.device(device):
            return paged_key_weights(q, k_cache, page_table, cache_lens, weights, k_scale=k_scale, scale=scale,
                                     cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, last=last, row_indices=row_indices)
    nbytes = workspace_bytes(batch, q_heads, kv_heads, seq_len, dim, page_size, max_pages, n_seqs, int(max_seqlen),
                             int(last or 0))
    work = q.new_empty((nbytes + 1) // 2)
    _cache_lib.check("fd_paged_key_weights", _cache_lib.lib().fd_paged_key_weights(
        q_ptr, cache, weights.data_ptr(), q_strides, w_strides, rows, index, batch,
        q_heads, seq_len, float(scale), int(last or 0), cu_ptr, n_seqs, int(max_seqlen), work.data_ptr(), nbytes,
        _cache_lib.raw_stream(device)))


def paged_kv_evict(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    weights: torch.Tensor,
    new_table: torch.Tensor,
    keep: int,
    *,
    recent: int = 0,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    weights_out: torch.Tensor | None = None,
    row_indices: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    if k_cache.ndim != 4:
        raise ValueError("k_cache and v_cache must be [n_pages, Hkv, page_size, D] of one shape")
    if page_table.ndim != 2 or page_table.shape[0] < 1:
        raise ValueError("page_table must be int32 [requests, max_pages], of one request or more")
    if cache_lens is None:
        raise ValueError("cache_lens is required")
    keep, recent = int(keep), int(recent)
    if not 1 <= keep < 1 << 27 or not 0 <= recent <= keep:
        raise ValueError("keep must be positive and recent in [0, keep]")
    requests, max_pages = page_table.shape
    _, heads, page_size, _ = k_cache.shape
    device = k_cache.get_device()
    cache = check_cache(k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, requests)
    rows, w_strides = check_weights("weights", weights, heads, max_pages * page_size, device)
    if weights_out is None:
        weights_out = weights
    elif weights_out is not weights:
        check_weights("weights_out", weights_out, heads, max_pages * page_size, device)
        if weights_out.shape != weights.shape or weights_out.stride() != weights.stride():
            raise ValueError("weights and weights_out must have one shape and the same strides")
        gap = abs(weights.data_ptr() - weights_out.data_ptr()) // 4
        if 0 < gap <= sum((n - 1) * s for n, s in zip(weights.shape, weights.stride())):
            raise ValueError("weights and weights_out must be the same memory or not overlap")
    new_shape, new_strides = new_table.shape, new_table.stride()
    if (len(new_shape) != 2 or new_shape[0] != requests or new_table.dtype is not torch.int32
            or new_table.get_device() != device or new_strides[1] != 1 or new_shape[1] * page_size < keep):
        raise ValueError(f"new_table must be int32 [{requests}, n] on the cache's device, its rows contiguous, and hold {keep} keys")
    if requests * heads * keep >= 1 << 27:
        raise ValueError("requests * Hkv * keep must be below 2^27")
    index = check_row_indices(row_indices, requests, rows, device)
    if _cache_lib.current_device() != device:
        with torch.cuda.device(device):
            return paged_kv_evict(k_cache, v_cache, page_table, cache_lens, weights, new_table, keep, recent=recent,
                                  k_scale=k_scale, v_scale=v_scale, weights_out=weights_out, row_indices=row_indices)
    kept, new_lens = page_table.new_empty((requests, heads, keep)), page_table.new_empty(requests)
    _cache_lib.check("fd_paged_kv_evict", _cache_lib.lib().fd_paged_kv_evict(
        cache, weights.data_ptr(), weights_out.data_ptr(), w_strides, rows, index,
        new_table.data_ptr(), new_strides[0], new_shape[1], requests, keep, recent, kept.data_ptr(),
        new_lens.data_ptr(), _cache_lib.raw_stream(device)))
    return kept, new_lens
