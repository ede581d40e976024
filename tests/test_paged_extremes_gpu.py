"""The ends of what a paged cache holds."""
from __future__ import annotations

import pytest
import torch

from cache_reference import pow2
from helpers import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_largest_values_come_back_finite(dim):
    """Every finite bf16 value from 1.5 2^127 on, alone in its row or beside smaller ones: E4M3 pages give it back
    within half a step of its code, and finite; infinities beside them stay."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    announce(f"e4m3 pages, largest values x {dim}")
    bits = torch.arange(0x7f40, 0x7f80, dtype=torch.int32).to(torch.int16)
    top = bits.view(torch.bfloat16).cuda()
    n = top.numel()
    x = torch.zeros((n, dim), dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, dim - 1], x[:, 7] = top, -top, top * 0.5
    odd = x.clone()
    odd[:, 3], odd[:, 4], odd[:, 5] = float("inf"), -float("inf"), float("nan")
    kc = torch.zeros((2, 1, 64, dim), dtype=torch.float8_e4m3fn, device="cuda")
    vc = torch.zeros_like(kc)
    ks, vs = (torch.full((2, 1, 64), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    paged_kv_write(x[None, None], odd[None, None], kc, vc, table, lens, k_scale=ks, v_scale=vs)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    k, v = (t[0, 0].double() for t in paged_kv_read(kc, vc, table, cu, n, k_scale=ks, v_scale=vs))
    assert torch.isfinite(k).all()
    # half a step of a code in [2^e, 2^(e + 1)) is 2^(e - 4): at most 2^-4 of the value
    assert ((k - x.double()).abs() <= 2.0 ** -4 * x.double().abs()).all()
    plain = torch.ones(dim, dtype=torch.bool, device="cuda")
    plain[3:6] = False
    assert torch.equal(v[:, plain], k[:, plain]) and torch.isnan(v[:, 5]).all()
    high = pow2(vs[1, 0, :n]) * 448 > torch.finfo(torch.bfloat16).max
    assert high.any() and (v[high, 3] == float("inf")).all() and (v[high, 4] == -float("inf")).all()
    assert torch.isfinite(v[~high, 3]).all()
