"""Bookkeeping of DeciderCache: pages, forks, steps and refusals (no GPU)."""
from __future__ import annotations

import pytest
import torch

from fastdecisions_amd.decider_cache import DeciderCache
from fastdecisions_amd.model import TINY


def make(**kw):
    return DeciderCache(TINY, **(dict(requests=4, tokens=200, max_tokens=100, page_size=16, device="cpu") | kw))


def test_shapes_and_layers():
    c = make(kv_dtype=torch.float8_e4m3fn)
    assert c.k.shape == c.v.shape == (1, 13 + 4, 1, 16, 64) and c.k_scale.shape == (1, 17, 1, 16)
    assert c.conv.shape == (3, 4, 3, 768) and c.delta.shape == (3, 4, 2, 128, 128)
    assert c.attention_layer(3)[0].shape == (17, 1, 16, 64) and c.linear_layer(2)[1].shape == (4, 2, 128, 128)
    with pytest.raises(KeyError):
        c.attention_layer(0)


def test_steps():
    c = make()
    a, b = c.open(), c.open()
    s = c.step([b, a], [20, 3])
    assert s.cu_seqlens.tolist() == [0, 20, 23] and s.cache_lens.tolist() == [20, 3]
    assert s.state_indices.tolist() == [b, a] and s.positions.tolist() == [[*range(20), 0, 1, 2]]
    assert s.max_new == 20 and s.last_rows == [19, 22] and s.page_table.shape == (2, 7)
    held = s.page_table.tolist()
    assert sum(p >= 0 for p in held[0]) == 2 and sum(p >= 0 for p in held[1]) == 1
    s2 = c.step([a], [14])
    assert s2.cache_lens.tolist() == [17] and s2.positions.tolist() == [[*range(3, 17)]]
    assert s2.page_table[0, 0] == held[1][0] and s2.page_table[0, 1] >= 0
    tensors = [t.data_ptr() for t in (s2.cu_seqlens, s2.cache_lens, s2.page_table, s2.positions)]
    assert s2.again() is s2 and s2.cache_lens.tolist() == [31] and s2.positions.tolist() == [[*range(17, 31)]]
    assert tensors == [t.data_ptr() for t in (s2.cu_seqlens, s2.cache_lens, s2.page_table, s2.positions)]
    assert c.length(a) == 31 and c.length(b) == 20


def test_forks_share_whole_pages():
    c = make()
    a = c.open()
    c.step([a], [40])                                     # two whole pages and half of one
    c.k.uniform_()
    c.conv[:, a], c.delta[:, a] = 3.0, 5.0
    b = c.fork(a)
    sa, sb = c._pages[a], c._pages[b]
    assert sa[:2] == sb[:2] and sa[2] != sb[2] and c.length(b) == 40
    assert torch.equal(c.k[:, sa[2]], c.k[:, sb[2]]) and (c.conv[:, b] == 3.0).all() and (c.delta[:, b] == 5.0).all()
    free = len(c._free_pages)
    c.close(a)
    assert len(c._free_pages) == free + 1                  # its own last page; the others are b's too
    c.close(b)
    assert len(c._free_pages) == c.n_pages and c._users == [0] * c.n_pages
    d = c.open()
    assert (c.conv[:, d] == 0).all() and (c.delta[:, d] == 0).all() and c.length(d) == 0
    c.step([d], [32])
    e = c.fork(d)                                          # nothing partly filled: all pages shared
    assert c._pages[e] == c._pages[d]
    c.step([e], [1])
    assert c._pages[e][:2] == c._pages[d] and len(c._pages[e]) == 3


def test_refusals_leave_the_cache_as_it_was():
    c = make()
    a = c.open()
    for bad in (dict(requests=0), dict(tokens=0), dict(page_size=24), dict(kv_dtype=torch.float16)):
        with pytest.raises(ValueError):
            make(**bad)
    for slots, new in (([], []), ([a], [0]), ([a], [1, 2]), ([a, a], [1, 1]), ([a + 1], [1]), ([-1], [1])):
        with pytest.raises(ValueError):
            c.step(slots, new)
    with pytest.raises(RuntimeError, match="per request"):
        c.step([a], [113])
    others = [c.open() for _ in range(3)]
    with pytest.raises(RuntimeError, match="are open"):
        c.open()
    with pytest.raises(RuntimeError, match="are open"):
        c.fork(a)
    with pytest.raises(RuntimeError, match="free pages"):
        c.step([a, *others], [100] * 4)
    assert c.length(a) == 0 and len(c._free_pages) == c.n_pages
    c.close(a)
    with pytest.raises(ValueError):
        c.close(a)
    with pytest.raises(ValueError):
        c.fork(a)
