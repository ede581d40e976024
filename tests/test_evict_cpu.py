"""What the entry points for key weights and eviction refuse (no GPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from fastdecisions_amd import _cache_lib, _lib
from test_paged_cache_cpu import FAKE, cache

INV, ALIGN, UNS = _lib.FD_ERR_INVALID_ARGUMENT, _lib.FD_ERR_ALIGNMENT, _lib.FD_ERR_UNSUPPORTED


def test_key_weights_refuse_bad_arguments():
    lib = _cache_lib.lib()
    s4, odd = (ctypes.c_int64 * 4)(512, 128, 512, 1), (ctypes.c_int64 * 4)(512, 128, 500, 1)
    s2 = (ctypes.c_int64 * 2)(512, 128)

    def weigh(change=None, **kw):
        a = dict(q=FAKE, w=FAKE, qs=s4, ws=s2, rows=8, idx=None, batch=1, hq=16, t=1, scale=0.1, last=0, cu=None, n=0, top=None,
                 work=FAKE, size=1 << 40) | kw
        c = cache(**(change or {}))
        return lib.fd_paged_key_weights(a["q"], ctypes.byref(c), a["w"], a["qs"], a["ws"], a["rows"], a["idx"], a["batch"],
                                        a["hq"], a["t"], a["scale"], a["last"], a["cu"], a["n"],
                                        a["t"] if a["top"] is None else a["top"], a["work"], a["size"], None)
    assert weigh(q=None) == INV and weigh(w=None) == INV and weigh(hq=6) == INV and weigh(scale=0.0) == INV
    assert weigh(scale=float("nan")) == INV and weigh(last=-1) == INV and weigh(top=2) == INV
    assert weigh(q=FAKE + 2) == ALIGN and weigh(qs=odd) == ALIGN
    assert weigh(cu=FAKE) == INV and weigh(n=2) == INV and weigh(cu=FAKE, n=2, batch=2) == INV
    assert weigh(rows=0) == INV and weigh(batch=9) == INV and weigh(ws=(ctypes.c_int64 * 2)(-1, 128)) == INV
    assert weigh(work=None) == INV and weigh(size=100) == INV and weigh(work=FAKE + 4) == INV
    assert weigh(batch=1 << 15, t=1 << 15, rows=1 << 15) == UNS and weigh(hq=4 * 2049) == UNS
    assert weigh(dict(dtype=9)) == INV and weigh(dict(head_dim=96)) == UNS and weigh(dict(cache_lens=None)) == INV
    assert weigh(batch=0) == _lib.FD_OK and weigh(t=0) == _lib.FD_OK
    assert b"fd_paged_key_weights" in lib.fd_cache_last_error()
    size = lib.fd_paged_key_weights_workspace_bytes
    assert size(1, 16, 3, 1, 128, 16, 4, 0, 1, 0) == INV and size(1, 16, 4, 1, 128, 16, 4, 0, 2, 0) == INV
    assert size(1, 16, 4, 1, 128, 16, 4, 0, 1, -1) == INV and size(1, 16, 4, 1, 128, 16, 0, 0, 1, 0) == INV
    assert size(1, 16, 4, 1, 96, 16, 4, 0, 1, 0) == UNS and size(1, 16, 4, 1, 128, 16, 4, 0, 1, 0) > 0
    # kept scores stay within a bound, whatever the page table's width
    assert size(64, 16, 4, 1, 128, 64, 1 << 20, 0, 1, 0) < 1 << 29 and size(1, 16, 4, 131072, 128, 64, 2048, 0, 131072, 0) < 1 << 29


def test_evict_refuses_bad_arguments():
    lib = _cache_lib.lib()
    s2 = (ctypes.c_int64 * 2)(512, 128)

    def evict(change=None, **kw):
        a = dict(w=FAKE, out=FAKE, ws=s2, rows=8, idx=None, table=FAKE, pages=4, n=2, keep=50, recent=5, kept=FAKE, lens=FAKE) | kw
        c = cache(**(change or {}))
        return lib.fd_paged_kv_evict(ctypes.byref(c), a["w"], a["out"], a["ws"], a["rows"], a["idx"], a["table"], a["pages"],
                                     a["pages"], a["n"], a["keep"], a["recent"], a["kept"], a["lens"], None)
    for name in ("w", "out", "ws", "table", "kept", "lens"):
        assert evict(**{name: None}) == INV, name
    assert evict(keep=0) == INV and evict(recent=51) == INV and evict(recent=-1) == INV and evict(n=-1) == INV
    assert evict(keep=65) == INV and evict(pages=0) == INV and evict(rows=1) == INV and evict(ws=(ctypes.c_int64 * 2)(512, -1)) == INV
    assert evict(n=1 << 22, rows=1 << 22) == UNS and evict(n=1 << 19, rows=1 << 19, keep=1 << 10, pages=1 << 6) == UNS
    assert evict(dict(cache_lens=None)) == INV and evict(dict(page_size=8)) == UNS and evict(dict(k=FAKE + 8)) == ALIGN
    assert evict(n=0) == _lib.FD_OK
    assert b"fd_paged_kv_evict" in lib.fd_cache_last_error()


def test_tensors_that_do_not_fit_are_refused():
    from fastdecisions_amd.paged_evict_kernel import check_row_indices, check_weights, paged_key_weights, paged_kv_evict
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, w = torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16), torch.zeros((1, 2, 32))
    with pytest.raises(ValueError, match="CUDA device"):
        paged_key_weights(q, k, table, lens, w)
    with pytest.raises(ValueError, match="multiple of its heads"):
        paged_key_weights(q[:, :3], k, table, lens, w)
    with pytest.raises(ValueError, match="last must be"):
        paged_key_weights(q, k, table, lens, w, last=0)
    with pytest.raises(ValueError, match="scale must be positive"):
        paged_key_weights(q, k, table, lens, w, scale=-1.0)
    with pytest.raises(ValueError, match="cache_lens is required"):
        paged_key_weights(q, k, table, None, w)
    with pytest.raises(ValueError, match="CUDA device"):
        paged_kv_evict(k, k, table, lens, w, table, 8)
    for kw in (dict(keep=0), dict(keep=8, recent=9), dict(keep=8, recent=-1), dict(keep=1 << 27)):
        with pytest.raises(ValueError, match="keep must be"):
            paged_kv_evict(k, k, table, lens, w, table, **kw)
    with pytest.raises(ValueError, match="one request or more"):
        paged_kv_evict(k, k, table[:0], lens[:0], w, table[:0], 8)
    check_weights("w", w, 2, 32, -1)
    for bad in (w[:, :1], w.double(), w[:, :, :31], w[0], w.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError, match="at least 32"):
            check_weights("w", bad, 2, 32, -1)
    for same in (torch.zeros((1, 2, 32)).expand(3, -1, -1), torch.zeros((1, 1, 32)).expand(-1, 2, -1),
                 torch.zeros(200).as_strided((2, 2, 32), (40, 32, 1))):
        with pytest.raises(ValueError, match="same memory"):
            check_weights("w", same, 2, 32, -1)
    check_weights("w", torch.zeros((2, 3, 32)).transpose(0, 1), 2, 32, -1)
    assert check_row_indices(None, 2, 2, -1) is None
    for idx, n in ((None, 3), (torch.zeros(2, dtype=torch.int32), 3), (torch.zeros(3, dtype=torch.int64), 3),
                   (torch.zeros(6, dtype=torch.int32)[::2], 3)):
        with pytest.raises(ValueError):
            check_row_indices(idx, n, 2, -1)
