"""What the entry points refuse of a 4-bit cache, and the test oracle's own rule (no GPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from e2m1_reference import VALUES, codes, hold, pack, values
from fastdecisions_amd import _cache_lib, _lib
from test_paged_cache_cpu import FAKE, cache


def cache4(**kw):
    strides = (ctypes.c_int64 * 3)(4 * 16 * 64, 16 * 64, 64)
    scales = (ctypes.c_int64 * 2)(4 * 16 * 4, 16 * 4)
    return cache(**(dict(dtype=_cache_lib.FD_DTYPE_E2M1, k_strides=strides, v_strides=strides, k_scale=FAKE, v_scale=FAKE,
                         k_scale_strides=scales, v_scale_strides=scales) | kw))


@pytest.mark.parametrize("change, code", [
    (dict(k_scale=None), "INVALID_ARGUMENT"), (dict(v_scale=None), "INVALID_ARGUMENT"),
    (dict(k_scale=FAKE + 2), "ALIGNMENT"), (dict(v_scale=FAKE + 1), "ALIGNMENT"), (dict(k=FAKE + 8), "ALIGNMENT"),
    (dict(k_scale_strides=(ctypes.c_int64 * 2)(258, 64), v_scale_strides=(ctypes.c_int64 * 2)(258, 64)), "ALIGNMENT"),
    (dict(k_scale_strides=(ctypes.c_int64 * 2)(256, 66), v_scale_strides=(ctypes.c_int64 * 2)(256, 66)), "ALIGNMENT"),
    (dict(v_scale_strides=(ctypes.c_int64 * 2)(256, 128)), "UNSUPPORTED"),
    (dict(k_strides=(ctypes.c_int64 * 3)(4096, 1024, 40), v_strides=(ctypes.c_int64 * 3)(4096, 1024, 40)), "ALIGNMENT"),
    (dict(dtype=4), "INVALID_ARGUMENT")])
def test_a_bad_4_bit_cache_is_refused(change, code):
    lib = _cache_lib.lib()
    want = getattr(_lib, "FD_ERR_" + code)
    s4, s2, c = (ctypes.c_int64 * 4)(512, 128, 512, 1), (ctypes.c_int64 * 2)(128, 512), cache4(**change)
    assert lib.fd_paged_kv_write(FAKE, FAKE, s4, s4, ctypes.byref(c), 1, 1, None, 0, None) == want
    assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, 1, FAKE, 1, None) == want
    assert lib.fd_paged_gqa_fwd(FAKE, ctypes.byref(c), None, FAKE, s4, None, s4, 1, 16, 1, 0.1, None, 0, 1, FAKE, 1 << 40,
                                None) == want


def test_a_good_4_bit_cache_is_not():
    lib, c = _cache_lib.lib(), cache4()
    s4, s2 = (ctypes.c_int64 * 4)(512, 128, 512, 1), (ctypes.c_int64 * 2)(128, 512)
    assert lib.fd_paged_kv_write(FAKE, FAKE, s4, s4, ctypes.byref(c), 0, 1, None, 0, None) == _lib.FD_OK
    assert lib.fd_paged_kv_read(ctypes.byref(c), FAKE, FAKE, s2, s2, 0, FAKE, 1, None) == _lib.FD_OK


def test_4_bit_tensors_of_the_host_are_refused():
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    k = torch.zeros((4, 2, 16, 32), dtype=torch.uint8).view(torch.float4_e2m1fn_x2)
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA device"):
        paged_kv_write(x, x, k, k, table, lens)
    with pytest.raises(ValueError, match="heads and head dimension"):
        paged_kv_write(x[..., :32], x[..., :32], k, k, table, lens)
    with pytest.raises(ValueError, match="CUDA device"):
        paged_kv_read(k, k, table, torch.tensor([0, 4], dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="head dimension"):
        paged_gqa_attention(x[..., :32], k, k, table, lens)
    with pytest.raises(ValueError, match="CUDA device"):
        paged_gqa_attention(x, k, k, table, lens)


def test_the_oracle_holds_by_its_definition():
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn((50, 64), generator=gen) * torch.exp2(torch.randint(-9, 9, (50, 1), generator=gen).float())).double()
    code, scale = hold(x)
    back = values(pack(code), scale)
    assert torch.equal(codes(pack(code)), code)
    step = torch.exp2(scale.double() - 127).repeat_interleave(32, -1)
    # the nearest of the codes' values, and half a scale would not hold the block's largest
    grid = torch.tensor([*VALUES, *(-v for v in VALUES)]).double()
    assert torch.equal((x - back).abs(), ((x / step)[..., None] - grid).abs().amin(-1) * step)
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1) / torch.exp2(scale.double() - 127)
    assert (top <= 6).all() and (top > 3).all()
    tie = torch.zeros(1, 32, dtype=torch.float64)
    tie[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    assert values(pack(hold(tie)[0]), hold(tie)[1])[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
