"""Eviction on the GPU against its definition: which keys stay, and every byte of the cache afterwards."""
from __future__ import annotations

import math

import pytest
import torch

from helpers import announce
from test_key_weights_gpu import FORMATS, make
from test_paged_cache_gpu import ints

pytestmark = pytest.mark.gpu


def raw(t):
    return t.view(torch.int16 if t.dtype == torch.bfloat16 else torch.uint8)


def chosen(w, length, keep, recent):
    """The kept keys of one head, in order: plain Python on its weights."""
    left = min(length, keep)
    recent = min(recent, left)
    fixed = length - recent
    value = [-math.inf if math.isnan(x) else x for x in w[:fixed]]
    nan = [math.isnan(x) for x in w[:fixed]]
    best = sorted(range(fixed), key=lambda j: (nan[j], -value[j], j))[:left - recent]
    return sorted(best) + list(range(fixed, length))


def check(held, lens, keep, recent, heads, dim, page, seed, *, weights=None, index=None, in_place=False, absent=(), lost=()):
    from fastdecisions_amd.paged_evict_kernel import paged_kv_evict
    need = -(-keep // page)
    c, _ = make(held, [*lens, need * page * len(lens)], page, heads, dim, seed)  # the last request's pages become the new ones
    table, pool = c["table"][:len(lens)].clone(), c["k"].shape[0]
    new_table = c["table"][len(lens), :need * len(lens)].reshape(len(lens), need).clone()
    for r, at in absent:
        table[r, at] = pool + 3
    for r, at in lost:
        new_table[r, at] = -1
    width = table.shape[1] * page
    gen = torch.Generator(device="cuda").manual_seed(seed + 2)
    index = list(range(len(lens))) if index is None else index
    w = torch.exp(torch.randn((len(lens) + 2, heads, width + 3), generator=gen, device="cuda"))
    if weights is not None:
        w = weights(w, gen)
    want = {name: raw(c[name]).clone() for name in ("k", "v", "ks", "vs") if c[name] is not None}
    before = {name: t.clone() for name, t in want.items()}
    want_w = w.clone() if in_place else torch.full_like(w, 7.0)
    want_kept = torch.full((len(lens), heads, keep), -1, dtype=torch.int32)
    for r, length in enumerate(lens):
        slot = index[r] if 0 <= index[r] < w.shape[0] and index[r] not in index[:r] else None
        for h in range(heads):
            mine = chosen(w[slot, h].tolist() if slot is not None else [0.0] * length, length, keep, recent)
            n = len(mine)
            want_kept[r, h, :n] = torch.tensor(mine, dtype=torch.int32)
            old = torch.tensor(mine, device="cuda", dtype=torch.long)
            if slot is not None:
                want_w[slot, h, :n] = w[slot, h, old]
                want_w[slot, h, n:length] = 0.0
            at = torch.arange(n, device="cuda")
            src, dst = table[r].long()[old // page], new_table[r].long()[at // page]
            live = (dst >= 0) & (dst < pool)
            there = (src >= 0) & (src < pool)
            for name, t in want.items():
                rows = before[name][src.clamp(0, pool - 1), h, old % page]
                rows[~there] = 127 if name in ("ks", "vs") else 0
                t[dst[live], h, (at % page)[live]] = rows[live]
    got_w = w if in_place else torch.full_like(w, 7.0)
    kept, left = paged_kv_evict(c["k"], c["v"], table, ints(lens), w, new_table, keep, recent=recent, k_scale=c["ks"],
                                v_scale=c["vs"], weights_out=None if in_place else got_w, row_indices=ints(index))
    assert left.tolist() == [min(n, keep) for n in lens]
    assert torch.equal(kept.cpu(), want_kept)
    assert torch.equal(got_w.view(torch.int32), want_w.view(torch.int32))
    for name, t in want.items():
        assert torch.equal(raw(c[name]), t), name


@pytest.mark.parametrize("held", FORMATS)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("heads,dim,page", [(4, 128, 16), (2, 256, 64), (3, 64, 256), (1, 128, 32)])
def test_keys_stay_by_weight(heads, dim, page, in_place, held):
    announce(f"evict, {heads} x {dim}, page {page}, in place {in_place}, {held}")
    check(held, [1, 2, 99, 100, 101, 133, 1000, 0, 2049, 5000], 100, 20, heads, dim, page, dim + page, in_place=in_place)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (37, 0), (37, 37), (300, 1), (4097, 100), (6000, 0)])
def test_every_share_of_recent_keys(keep, recent):
    announce(f"evict, keep {keep}, recent {recent}")
    check("bf16", [4096, 300, 6000, 38, 37, 12345], keep, recent, 2, 64, 64, keep, in_place=True)


def some_equal(w, gen):
    return (w * 2).round() / 2


def zeros_and_odd(w, gen):
    w = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.6, 0.0, w)
    pick = torch.randint(0, 40, w.shape, generator=gen, device="cuda")
    for i, v in enumerate((math.nan, math.inf, -math.inf, -0.0, -1.5, 1e-45, 3e38)):
        w = w.masked_fill(pick == i, v)
    return w.contiguous()


@pytest.mark.parametrize("weights", [some_equal, zeros_and_odd, lambda w, gen: torch.zeros_like(w),
                                     lambda w, gen: torch.full_like(w, math.nan)])
@pytest.mark.parametrize("in_place", [False, True])
def test_equal_and_odd_weights(weights, in_place):
    """Ties go to the lowest key; NaN stays behind everything, infinities are numbers."""
    announce("evict, equal and odd weights")
    check("e2m1", [700, 5000, 9000, 65], 64, 7, 2, 64, 16, 3, weights=weights, in_place=in_place)


def test_rows_and_pages_that_are_not_there():
    """A request without a row of weights keeps its first keys; keys on no page become zeros; no page, no write."""
    announce("evict, rows and pages that are not there")
    check("e4m3", [100, 200, 300, 400], 48, 16, 2, 128, 16, 4, index=[5, 1, 5, -1], absent=[(0, 1), (1, 12), (2, 0)],
          lost=[(0, 0), (3, 2)])


@pytest.mark.parametrize("held", FORMATS)
def test_many_requests(held):
    announce(f"evict, 150 requests, {held}")
    check(held, [1 + (i * 37) % 300 for i in range(150)], 64, 16, 2, 64, 16, 5, in_place=True)


def test_a_long_request():
    announce("evict, 150000 keys")
    check("e2m1", [150001, 70000], 9001, 333, 1, 64, 256, 6)


def test_long_requests_in_place():
    """Beyond the weights that stay in registers, their moves overtake no load; equal weights at the border."""
    announce("evict in place, 16384 to 70000 keys")
    check("e2m1", [70000, 16385, 16384, 40000], 1000, 50, 2, 64, 64, 7, weights=some_equal, in_place=True)
    check("bf16", [33000, 20000], 18000, 0, 1, 64, 256, 8, in_place=True)
