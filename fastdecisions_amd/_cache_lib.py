"""ctypes binding of ``libfd_cache.so`` (the C ABI in ``include/fd_cache.h``): the
kernels that continue a request from its caches.  Loaded after torch and without a
fallback, as ``libfd_kernels.so`` is (``_lib``); ``FD_CACHE_LIB`` names another build
of it to load."""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch

from . import _lib

LIB_PATH = Path(os.environ.get("FD_CACHE_LIB", Path(__file__).resolve().parent / "libfd_cache.so"))

FD_DTYPE_E4M3 = 2

_p, _i, _i64, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_i64s = ctypes.POINTER(ctypes.c_int64)


class PagedCache(ctypes.Structure):
    """``fd_paged_cache``."""
    _fields_ = [("k", _p), ("v", _p), ("k_scale", _p), ("v_scale", _p),
                ("k_strides", _i64 * 3), ("v_strides", _i64 * 3),
                ("k_scale_strides", _i64 * 2), ("v_scale_strides", _i64 * 2),
                ("page_table", _p), ("table_stride", _i64), ("cache_lens", _p),
                ("n_pages", ctypes.c_int32), ("page_size", ctypes.c_int32), ("max_pages", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


_cache = ctypes.POINTER(PagedCache)
SIGNATURES = {
    "fd_cache_abi_version": (_i, []),
    "fd_cache_last_error": (ctypes.c_char_p, []),
    "fd_paged_kv_write": (_i, [_p, _p, _i64s, _i64s, _cache, _i, _i, _p, _i, _p]),
    "fd_paged_kv_read": (_i, [_cache, _p, _p, _i64s, _i64s, _i64, _p, _i, _p]),
    "fd_paged_gqa_fwd": (_i, [_p, _cache, _p, _p, _i64s, _i64s, _i64s, _i, _i, _i, _f, _p, _i, _i, _p, _i64, _p]),
    "fd_paged_gqa_workspace_bytes": (_i64, [_i] * 9),
}

_LIB = None


def lib() -> ctypes.CDLL:
    """Load (once) and return the cache library; raise if it is unavailable."""
    global _LIB
    if _LIB is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"HIP cache library not found at {LIB_PATH}; build it first "
                "(python -c 'import __graft_entry__ as g; g.build()' or python -m fastdecisions_amd._build)")
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = handle
    return _LIB


def check(name: str, code: int) -> None:
    if code < 0:
        raise _lib.KernelError(name, code, lib().fd_cache_last_error().decode(errors="replace"))


def strides(t: torch.Tensor, n: int) -> ctypes.Array:
    """The first n strides of t in elements."""
    return (_i64 * n)(*t.stride()[:n])
