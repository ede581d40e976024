"""The cache library's C ABI and the refusals of the paged cache's entry points (no GPU)."""
from __future__ import annotations

import ctypes
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from fastdecisions_amd import _build, _cache_lib, _lib

import test_isa_cpu
from test_isa_cpu import (test_a_wait_state_between_m0_and_the_copy_that_reads_it,  # noqa: F401
                          test_no_asm_leaves_a_global_load_into_registers_in_flight,
                          test_registers_of_asm_lds_reads_are_untouched_until_their_wait)

HEADER = ROOT / "include" / "fd_cache.h"
FAKE = 1 << 20  # 16-byte aligned, never dereferenced: validation fails first


@pytest.fixture(scope="module")
def kernels():
    """The hazards that the other library's sources are checked for, in this one's."""
    request = type("Request", (), {"param": "paged_gqa.hip"})
    get = test_isa_cpu.kernels
    get = get.__wrapped__ if hasattr(get, "__wrapped__") else get.__pytest_wrapped__.obj
    with pytest.MonkeyPatch.context() as m:
        m.setattr(_build, "DEVICE_FLAGS", _build.DEVICE_FLAGS + _build.EXTRA_FLAGS["paged_gqa.hip"])
        return get(request)


def declared():
    return set(re.findall(r"FD_API\s+[\w\s\*]+?\b(fd_\w+)\s*\(", HEADER.read_text()))


def test_library_exports_what_its_header_declares():
    lib = _cache_lib.lib()
    out = subprocess.run(["nm", "-D", "--defined-only", str(_cache_lib.LIB_PATH)], capture_output=True, text=True,
                         check=True).stdout
    assert {line.split()[-1] for line in out.splitlines() if " T " in line} == declared() == set(_cache_lib.SIGNATURES)
    version = int(re.search(r"#define FD_CACHE_ABI_VERSION (\d+)", HEADER.read_text()).group(1))
    assert lib.fd_cache_abi_version() == version
    assert not set(_build.SOURCES) & set(_build.CACHE_SOURCES)


def cache(**kw):
    c = _cache_lib.PagedCache()
    c.k = c.v = c.page_table = c.cache_lens = FAKE
    c.k_strides[:] = c.v_strides[:] = (4 * 16 * 128, 16 * 128, 128)
    c.table_stride, c.n_pages, c.page_size, c.max_pages, c.kv_heads, c.head_dim = 8, 10, 16, 8, 4, 128
    c.dtype = _lib.FD_DTYPE_BF16
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change, code", [
    (dict(k=None), "INVALID_ARGUMENT"), (dict(page_table=None), "INVALID_ARGUMENT"),
    (dict(cache_lens=None), "INVALID_ARGUMENT"), (dict(head_dim=96), "UNSUPPORTED"), (dict(page_size=8), "UNSUPPORTED"),
    (dict(page_size=48), "UNSUPPORTED"), (dict(page_size=512), "UNSUPPORTED"), (dict(dtype=7), "INVALID_ARGUMENT"),
    (dict(dtype=2), "INVALID_ARGUMENT"), (dict(n_pages=0), "INVALID_ARGUMENT"), (dict(max_pages=0), "INVALID_ARGUMENT"),
    (dict(max_pages=1 << 27), "UNSUPPORTED"), (dict(k=FAKE + 8), "ALIGNMENT"),
    (dict(k_strides=(ctypes.c_int64 * 3)(4, 16 * 128, 128), v_strides=(ctypes.c_int64 * 3)(4, 16 * 128, 128)), "ALIGNMENT"),
    (dict(k_strides=(ctypes.c_int64 * 3)(8192, 2048, 1 << 20), v_strides=(ctypes.c_int64 * 3)(8192, 2048, 1 << 20)),
     "UNSUPPORTED"),
    (dict(k_strides=(ctypes.c_int64 * 3)(1 << 35, 2048, 128), v_strides=(ctypes.c_int64 * 3)(1 << 35, 2048, 128)),
     "UNSUPPORTED"),
    (dict(v_strides=(ctypes.c_int64 * 3)(8192, 2048, 256)), "UNSUPPORTED")])
def test_a_bad_cache_is_refused(change, code):
    lib = _cache_lib.lib()
    want = getattr(_lib, "FD_ERR_" + code)
    s4, c = (ctypes.c_int64 * 4)(512, 128, 512, 1), cache(**change)
    assert lib.fd_paged_kv_write(FAKE, FAKE, s4, s4, ctypes.byref(c), 1, 1, None, 0, None) == want
    assert b"fd_paged_kv_write" in lib.fd_cache_last_error()
    assert lib.fd_paged_gqa_fwd(FAKE, ctypes.byref(c), None, FAKE, s4, None, s4, 1, 16, 1, 0.1, None, 0, 1, FAKE, 1 << 40,
                                None) == want
    if "cache_lens" not in change:
        s2 = (ctypes.c_int64 * 2)(128, 512)
        assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, 1, FAKE, 1, None) == want


def test_bad_arguments_are_refused():
    lib = _cache_lib.lib()
    inv, align, uns = _lib.FD_ERR_INVALID_ARGUMENT, _lib.FD_ERR_ALIGNMENT, _lib.FD_ERR_UNSUPPORTED
    c = cache()
    s4 = (ctypes.c_int64 * 4)(512, 128, 512, 1)
    odd = (ctypes.c_int64 * 4)(512, 128, 500, 1)

    def gqa(**kw):
        a = dict(q=FAKE, gate=None, out=FAKE, qs=s4, gs=None, os=s4, batch=1, hq=16, t=1, scale=0.1, cu=None, n=0,
                 top=None, work=FAKE, size=1 << 40) | kw
        a["top"] = a["t"] if a["top"] is None else a["top"]
        return lib.fd_paged_gqa_fwd(a["q"], ctypes.byref(c), a["gate"], a["out"], a["qs"], a["gs"], a["os"], a["batch"],
                                    a["hq"], a["t"], a["scale"], a["cu"], a["n"], a["top"], a["work"], a["size"], None)
    assert gqa(q=None) == inv and gqa(hq=6) == inv and gqa(scale=0.0) == inv and gqa(scale=float("nan")) == inv
    assert gqa(q=FAKE + 2) == align and gqa(qs=odd) == align and gqa(gate=FAKE) == inv
    assert gqa(cu=FAKE) == inv and gqa(n=2) == inv and gqa(cu=FAKE, n=2, batch=2) == inv and gqa(top=2) == inv
    assert gqa(batch=1 << 15, t=1 << 15) == uns
    c.max_pages = 64
    assert gqa(work=None) == inv and gqa(size=100) == inv and gqa(work=FAKE + 4) == inv
    assert gqa(batch=0) == _lib.FD_OK and gqa(t=0) == _lib.FD_OK
    assert lib.fd_paged_kv_write(FAKE, FAKE, odd, s4, ctypes.byref(c), 1, 1, None, 0, None) == align
    assert lib.fd_paged_kv_write(FAKE, FAKE, s4, s4, ctypes.byref(c), 2, 1, FAKE, 3, None) == inv
    assert lib.fd_paged_kv_write(FAKE, FAKE, s4, s4, ctypes.byref(c), 0, 1, None, 0, None) == _lib.FD_OK
    s2 = (ctypes.c_int64 * 2)(128, 512)
    assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, 1, None, 1, None) == inv
    assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, -1, FAKE, 1, None) == inv
    assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, 0, FAKE, 1, None) == _lib.FD_OK
    assert lib.fd_paged_gqa_workspace_bytes(1, 16, 3, 1, 128, 16, 4, 0, 1) == inv
    assert lib.fd_paged_gqa_workspace_bytes(1, 16, 4, 1, 100, 16, 4, 0, 1) == uns
    assert lib.fd_paged_gqa_workspace_bytes(1, 16, 4, 1, 128, 16, 4, 0, 1) == 0  # too few keys to split
    assert lib.fd_paged_gqa_workspace_bytes(1, 16, 4, 1, 128, 16, 64, 0, 1) > 0


def test_tensors_that_do_not_fit_are_refused():
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA device"):
        paged_kv_write(x, x, k, k, table, lens)
    with pytest.raises(ValueError, match="heads and head dimension"):
        paged_kv_write(x[:, :1], x[:, :1], k, k, table, lens)
    with pytest.raises(ValueError, match="of one shape"):
        paged_kv_write(x, x[:, :, :, :32], k, k, table, lens)
    with pytest.raises(ValueError, match="CUDA device"):
        paged_kv_read(k, k, table, torch.tensor([0, 4], dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="multiple of its heads"):
        paged_gqa_attention(torch.zeros((1, 3, 1, 64), dtype=torch.bfloat16), k, k, table, lens)
    with pytest.raises(ValueError, match="scale must be positive"):
        paged_gqa_attention(x, k, k, table, lens, scale=-1.0)
    with pytest.raises(ValueError, match="cu_seqlens requires batch size 1"):
        paged_gqa_attention(x.expand(2, -1, -1, -1), k, k, table, lens, cu_seqlens=torch.zeros(3, dtype=torch.int32))


def test_a_write_of_no_tokens_is_refused():
    from fastdecisions_amd.paged_kv_kernel import paged_kv_write
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    x = torch.zeros((1, 2, 0, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be positive"):
        paged_kv_write(x, x, k, k, torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32))


def test_calls_larger_than_a_grid_are_refused():
    """A grid dimension's threads fit 32 bits."""
    lib, c, uns = _cache_lib.lib(), cache(), _lib.FD_ERR_UNSUPPORTED
    s4, s2 = (ctypes.c_int64 * 4)(512, 128, 512, 1), (ctypes.c_int64 * 2)(128, 512)
    assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, 1 << 30, FAKE, 1, None) == uns
    assert lib.fd_paged_kv_write(FAKE, FAKE, s4, s4, ctypes.byref(c), 1 << 15, 1 << 15, None, 0, None) == uns
    assert lib.fd_gated_delta_step(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None, 0, None, 1 << 22, 1, 16, 16, 128, 128,
                                   0.1, _lib.FD_DTYPE_BF16, 0, None, 0, None) == uns
    assert lib.fd_packed_conv_state(FAKE, 6144, FAKE, None, FAKE, FAKE, 1 << 26, None, FAKE, FAKE, FAKE, 1 << 26, 1, 2048,
                                    2048, 4, None, 0, _lib.FD_ACT_SILU, None) == uns


def test_more_query_heads_per_key_head_than_a_row_count_holds_are_refused():
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    lib = _cache_lib.lib()
    assert lib.fd_paged_gqa_workspace_bytes(1, 2048, 1, 1, 64, 16, 64, 0, 1) > 0
    assert lib.fd_paged_gqa_workspace_bytes(1, 2049, 1, 1, 64, 16, 64, 0, 1) == _lib.FD_ERR_UNSUPPORTED
    k = torch.zeros((4, 1, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="2048 query heads"):
        paged_gqa_attention(torch.zeros((1, 2049, 1, 64), dtype=torch.bfloat16), k, k,
                            torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32))


def test_state_operators_refuse_bad_arguments():
    lib = _cache_lib.lib()
    inv, align, uns = _lib.FD_ERR_INVALID_ARGUMENT, _lib.FD_ERR_ALIGNMENT, _lib.FD_ERR_UNSUPPORTED

    def step(**kw):
        a = dict(q=FAKE, out=FAKE, s=FAKE, so=FAKE, pool=2, idx=None, B=2, T=1, hk=2, hv=4, dk=128, dv=128, bd=0, cu=None,
                 n=0) | kw
        return lib.fd_gated_delta_step(a["q"], FAKE, FAKE, FAKE, FAKE, a["out"], a["s"], a["so"], a["pool"], a["idx"],
                                       a["B"], a["T"], a["hk"], a["hv"], a["dk"], a["dv"], 0.1, a["bd"], 1, a["cu"], a["n"],
                                       None)
    assert step(q=None) == inv and step(hv=3) == inv and step(dk=64) == uns and step(bd=2) == inv
    assert step(pool=1) == inv and step(pool=0, idx=FAKE) == inv and step(so=FAKE + 4) == align
    assert step(cu=FAKE) == inv and step(n=2) == inv and step(cu=FAKE, n=2, B=2) == inv
    assert step(B=1 << 16, T=1 << 15, pool=1 << 16) == uns and step(B=0) == _lib.FD_OK

    def conv(**kw):
        a = dict(x=FAKE, row=384, s=FAKE, so=FAKE, pool=2, idx=None, B=2, T=1, kd=128, vd=128, W=4, cu=None, n=0, act=1) | kw
        return lib.fd_packed_conv_state(a["x"], a["row"], FAKE, None, a["s"], a["so"], a["pool"], a["idx"], FAKE, FAKE, FAKE,
                                        a["B"], a["T"], a["kd"], a["vd"], a["W"], a["cu"], a["n"], a["act"], None)
    assert conv(x=None) == inv and conv(s=None) == inv and conv(kd=12) == inv and conv(W=1) == uns and conv(W=5) == uns
    assert conv(row=380) == align and conv(row=376) == align and conv(x=FAKE + 2) == align and conv(act=3) == inv
    assert conv(pool=1) == inv and conv(cu=FAKE) == inv and conv(n=1) == inv and conv(B=0) == _lib.FD_OK


def test_states_that_do_not_fit_are_refused():
    check = lambda *a: _cache_lib.check_states(*a, (2, 4), torch.float32, torch.device("cpu"))
    s, idx = torch.zeros((3, 2, 4)), torch.zeros(2, dtype=torch.int32)
    assert check(s, s, None, 3) == (3, None) and check(s, None, idx, 2)[0] == 3 and check(None, None, None, 5) == (0, None)
    for bad in ((s, s, None, 2), (s[:, :1], None, None, 3), (s.double(), None, None, 3), (s, s[:2], None, 3),
                (s.transpose(1, 2).contiguous().transpose(1, 2), None, None, 3), (None, None, idx, 2),
                (s, None, idx.long(), 2), (s, None, idx, 3)):
        with pytest.raises(ValueError):
            check(*bad)
    big = torch.zeros((6, 2, 4))
    with pytest.raises(ValueError, match="overlap"):
        check(big[:4], big[2:], None, 4)


def test_tensors_of_the_host_are_refused():
    from fastdecisions_amd.gated_delta_kernel import recurrent_gated_delta_rule
    from fastdecisions_amd.packed_conv_kernel import prep_qkv_state
    x = torch.zeros((1, 1, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be on CUDA"):
        recurrent_gated_delta_rule(x, x, x, torch.zeros((1, 1, 2)), torch.zeros((1, 1, 2)))
    with pytest.raises(ValueError, match="must be on CUDA"):
        prep_qkv_state(torch.zeros((1, 1, 384), dtype=torch.bfloat16), torch.zeros((384, 4), dtype=torch.bfloat16),
                       torch.zeros((1, 3, 384), dtype=torch.bfloat16))
