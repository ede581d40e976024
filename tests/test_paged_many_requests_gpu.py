"""Paged attention of more requests than a wavefront has lanes: packed, ragged, some without new tokens."""
from __future__ import annotations

import pytest

from helpers import announce
from test_paged_cache_gpu import check_attention, make_q, run_attention
from cache_reference import make_pages

pytestmark = pytest.mark.gpu


def sizes(count, top):
    """New and cached tokens of ``count`` requests: up to ``top`` new ones, none around the borders between rounds
    of 64 lanes and of the last request, prefixes from nothing to a few that are split over workgroups."""
    new = [1 + (i * 29) % top for i in range(count)]
    for i in (0, 63, 64, 127, count - 1):
        new[i] = 0
    cached = [(i * 67) % 350 for i in range(count)]
    for i, n in ((5, 5000), (62, 3333), (65, 6100), (126, 2047), (128, 4096)):
        cached[i] = n
    return new, [c + n for c, n in zip(cached, new)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("top", [1, 7, 16, 40])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
def test_packed_requests_beyond_64(hq, hkv, dim, top, fp8):
    """Four rows of a key head up to 160: tiles of 16, of 32 and of 128 rows, split and joined."""
    new, lens = sizes(140, top)
    announce(f"paged attention, 140 packed requests of up to {top} tokens, {hq}/{hkv} x {dim}, fp8 {fp8}")
    c = make_pages(lens, 16, hkv, dim, fp8, seed=30)
    q = make_q(new, hq, dim, 31)
    gate = make_q(new, hq, dim, 32)
    out = run_attention(c, q, lens, new, gate=gate)
    check_attention(c, q, out, lens, new, gate=gate)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,dim", [(64, 4, 128), (64, 8, 256), (128, 4, 64)])
@pytest.mark.parametrize("new,cached", [([1100], [200]), ([1, 1100, 30, 0], [5000, 0, 2000, 77])])
def test_more_row_tiles_than_places_for_parts(new, cached, hq, hkv, dim, fp8):
    """More row tiles than two rounds of workgroups: nothing is split, and no tile needs a place in the workspace."""
    announce(f"paged attention, {new} tokens x {hq}/{hkv} x {dim}, fp8 {fp8}")
    lens = [n + c for n, c in zip(new, cached)]
    c = make_pages(lens, 64, hkv, dim, fp8, seed=33)
    q = make_q(new, hq, dim, 34)
    out = run_attention(c, q, lens, new)
    check_attention(c, q, out, lens, new)
