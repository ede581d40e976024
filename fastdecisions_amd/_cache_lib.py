"""ctypes binding of ``libfd_cache.so`` (the C ABI in ``include/fd_cache.h``): the
kernels that continue a request from its caches.  Loaded after torch and without a
fallback, as ``libfd_kernels.so`` is (``_lib``); ``FD_CACHE_LIB`` names another build
of it to load."""
from __future__ import annotations

import ctypes
import os
import struct
from pathlib import Path

import torch

from . import _lib

LIB_PATH = Path(os.environ.get("FD_CACHE_LIB", Path(__file__).resolve().parent / "libfd_cache.so"))

FD_DTYPE_E4M3 = 2
FD_DTYPE_E2M1 = 3

# Strides and the cache struct are handed over as packed bytes (c_void_p takes them): building ctypes
# arrays and structures field by field costs microseconds a call, as much as a small launch.
_p, _i, _i64, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
pack2, pack4 = struct.Struct("2q").pack, struct.Struct("4q").pack
pack_cache = struct.Struct("4Q10qQqQ6i").pack  # the fields of fd_paged_cache in order


class PagedCache(ctypes.Structure):
    """``fd_paged_cache`` (``from_buffer_copy`` of the packed form)."""
    _fields_ = [("k", _p), ("v", _p), ("k_scale", _p), ("v_scale", _p),
                ("k_strides", _i64 * 3), ("v_strides", _i64 * 3),
                ("k_scale_strides", _i64 * 2), ("v_scale_strides", _i64 * 2),
                ("page_table", _p), ("table_stride", _i64), ("cache_lens", _p),
                ("n_pages", ctypes.c_int32), ("page_size", ctypes.c_int32), ("max_pages", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


SIGNATURES = {
    "fd_cache_abi_version": (_i, []),
    "fd_cache_last_error": (ctypes.c_char_p, []),
    "fd_paged_kv_write": (_i, [_p, _p, _p, _p, _p, _i, _i, _p, _i, _p]),
    "fd_paged_kv_read": (_i, [_p, _p, _p, _p, _p, _i64, _p, _i, _p]),
    "fd_paged_gqa_fwd": (_i, [_p, _p, _p, _p, _p, _p, _p, _i, _i, _i, _f, _p, _i, _i, _p, _i64, _p]),
    "fd_paged_gqa_workspace_bytes": (_i64, [_i] * 9),
    "fd_paged_key_weights": (_i, [_p, _p, _p, _p, _p, _i, _p, _i, _i, _i, _f, _i, _p, _i, _i, _p, _i64, _p]),
    "fd_paged_key_weights_workspace_bytes": (_i64, [_i] * 10),
    "fd_paged_kv_evict": (_i, [_p, _p, _p, _p, _i, _p, _p, _i64, _i, _i, _i, _i, _p, _p, _p]),
    "fd_gated_delta_step": (_i, [_p] * 8 + [_i, _p] + [_i] * 6 + [_f, _i, _i, _p, _i, _p]),
    "fd_packed_conv_state": (_i, [_p, _i64, _p, _p, _p, _p, _i, _p, _p, _p, _p] + [_i] * 5 + [_p, _i, _i, _p]),
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


current_device = torch._C._cuda_getDevice
raw_stream = torch._C._cuda_getCurrentRawStream


def check_states(state, state_out, state_indices, requests: int, shape: tuple, dtype, device) -> tuple[int, int | None]:
    """Validate a state pool ``[n, *shape]``, where it is written and the rows requests own in it;
    returns (rows of the pool, pointer of the indices)."""
    for name, t in (("state", state), ("state_out", state_out)):
        if t is None or (t is state and name == "state_out"):
            continue
        if t.shape[1:] != shape or t.dtype != dtype or t.device != device or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned {dtype} tensor [n, "
                             f"{', '.join(map(str, shape))}] on the inputs' device")
    pool = state if state is not None else state_out
    n_pool = 0 if pool is None else pool.shape[0]
    if state is not None and state_out is not None and state_out is not state:
        if state.shape != state_out.shape:
            raise ValueError("state and state_out must have one shape")
        a, b = state.data_ptr(), state_out.data_ptr()
        if a != b and abs(a - b) < state.numel() * state.element_size():
            raise ValueError("state and state_out must be the same memory or not overlap")
    if state_indices is None:
        if pool is not None and n_pool != requests:
            raise ValueError(f"Without state_indices the state has one row for each of the {requests} requests")
        return n_pool, None
    if n_pool < 1:
        raise ValueError("state_indices need a state")
    if (state_indices.shape != (requests,) or state_indices.dtype != torch.int32 or state_indices.device != device
            or not state_indices.is_contiguous()):
        raise ValueError(f"state_indices must be a contiguous int32 vector [{requests}] on the inputs' device")
    return n_pool, state_indices.data_ptr()
