"""Workspace of the paged attention (no GPU: the library computes it from the sizes)."""
from __future__ import annotations

import pytest

from fastdecisions_amd.paged_gqa_kernel import workspace_bytes

CUS = 256


@pytest.mark.parametrize("requests", [1, 64])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 128), (8, 2, 256), (16, 4, 64), (8, 8, 128)])
def test_long_pieces_take_no_more(hq, hkv, dim, requests):
    """Keys are split only where all items fit two rounds of workgroups, so parts are bounded by them: two rounds of at
    most two workgroups per CU, 128 rows of D + 2 words each, however many row tiles the tokens have."""
    bound = 256 + 2 * 2 * CUS * 128 * (dim + 2) * 4
    for tokens in (4096, 16384, 131072):
        got = workspace_bytes(1, hq, hkv, tokens, dim, 64, 2048, requests, tokens)
        assert 0 < got <= bound, (tokens, got)
    assert workspace_bytes(1, hq, hkv, 131072, dim, 64, 2048, requests, 131072) == \
        workspace_bytes(1, hq, hkv, 4096, dim, 64, 2048, requests, 4096)
