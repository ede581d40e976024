"""What a DeciderCache keeps track of when keys are evicted (no GPU: the kernels' op is replaced)."""
from __future__ import annotations

import pytest
import torch

from fastdecisions_amd import cached_ops
from fastdecisions_amd.decider_cache import DeciderCache
from fastdecisions_amd.model import TINY


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(cached_ops, "paged_kv_evict_op", lambda *a: seen.append(a))
    return seen


def make(**kw):
    return DeciderCache(TINY, **(dict(requests=3, tokens=200, max_tokens=100, page_size=16, key_weights=True, device="cpu") | kw))


def layers():
    return sum((i + 1) % TINY.full_attention_interval == 0 for i in range(TINY.num_hidden_layers))


def test_an_evicted_request_goes_on_where_it_stood(calls):
    c = make()
    a, b = c.open(), c.open()
    c.step([a, b], [90, 20])
    free = len(c._free_pages)
    c.evict([a, b], 24, recent=4)
    assert len(calls) == layers()
    k, v, table, lens, w, new_table, keep, recent, ks, vs, rows = calls[0]
    assert (table.shape, new_table.shape, lens.tolist(), rows.tolist(), keep, recent) == ((1, 6), (1, 2), [90], [a], 24, 4)
    assert w.shape == (3, TINY.num_key_value_heads, 7 * 16) and not set(table.flatten().tolist()) & set(new_table.flatten().tolist())
    assert c._pages[a] == new_table[0].tolist()
    assert (c.length(a), c.position(a), c.length(b), c.position(b)) == (24, 90, 20, 20)
    assert len(c._free_pages) == free + 6 - 2
    step = c.step([a, b], [3, 1])
    assert step.positions.tolist() == [[90, 91, 92, 20]] and step.cache_lens.tolist() == [27, 21]
    assert step.page_table[0, :3].tolist() == c._pages[a] + [-1] * (3 - len(c._pages[a]))
    step.cancel()
    assert (c.length(a), c.position(a), c.position(b)) == (24, 90, 20)
    again = c.step([a], [2])
    assert again.again().positions.tolist() == [[92, 93]] and c.length(a) == 28


def test_a_fork_of_an_evicted_request(calls):
    c = make()
    a = c.open()
    c.step([a], [70])
    c.weights[:, a] = 2.0
    f = c.fork(a)
    assert (c.weights[:, f] == 2.0).all()
    shared = list(c._pages[a][:4])
    c.evict([f], 40)
    assert c._pages[a][:4] == shared and all(c._users[p] == 1 for p in shared)   # the parent's alone again
    assert (c.length(a), c.length(f), c.position(f)) == (70, 40, 70)
    g = c.fork(f)
    assert (c.length(g), c.position(g)) == (40, 70)
    for s in (a, f, g):
        c.close(s)
    assert len(c._free_pages) == c.n_pages and c._users == [0] * c.n_pages
    n = c.open()
    assert c.position(n) == 0 and (c.weights[:, n] == 0).all()


def test_steps_made_before_are_refused(calls):
    c = make()
    a = c.open()
    step = c.step([a], [50])
    c.evict([a], 10)
    with pytest.raises(ValueError, match="evicted"):
        step.again()
    step.cancel()                      # nothing of it is left to take back
    assert c.length(a) == 10


def test_what_is_refused(calls):
    c = make()
    a = c.open()
    c.step([a], [100])
    for kw in (dict(keep=0), dict(keep=5, recent=6), dict(keep=5, recent=-1)):
        with pytest.raises(ValueError, match="keep must be"):
            c.evict([a], **kw)
    with pytest.raises(ValueError, match="appears once"):
        c.evict([a, a], 5)
    with pytest.raises(ValueError, match="no open request"):
        c.evict([a + 1], 5)
    with pytest.raises(RuntimeError, match="key_weights=True"):
        make(key_weights=False).evict([], 5)
    for bad in (dict(observe=0), dict(observe=4, key_weights=False)):
        with pytest.raises(ValueError, match="observe"):
            make(**bad)
    b = c.open()
    c.step([b], [90])                  # 16 pages in all, 13 taken
    with pytest.raises(RuntimeError, match="free pages"):
        c.evict([a], 70)
    assert c.length(a) == 100 and not calls
    c.evict([a], 100)                  # holds no more: nothing to do
    assert not calls


def test_an_eviction_that_fails_on_the_way(monkeypatch):
    c = make()
    a = c.open()
    c.step([a], [60])
    pages, free = list(c._pages[a]), len(c._free_pages)

    def fail(*a):
        raise RuntimeError("out of memory")
    monkeypatch.setattr(cached_ops, "paged_kv_evict_op", fail)
    with pytest.raises(RuntimeError, match="out of memory"):
        c.evict([a], 20)
    assert c._pages[a] == pages and len(c._free_pages) == free
    with pytest.raises(RuntimeError, match="only be closed"):
        c.step([a], [1])
    c.close(a)
    assert len(c._free_pages) == c.n_pages


def test_pools_of_4_bits():
    c = make(kv_dtype=torch.float4_e2m1fn_x2)
    d = TINY.head_dim
    assert c.k.dtype == torch.float4_e2m1fn_x2 and c.k.shape[-1] == d // 2
    assert c.k_scale.shape == (*c.k.shape[:4], d // 32) and (c.v_scale == 127).all()
    a = c.open()
    c.step([a], [20])
    c.k.view(torch.uint8)[:, c._pages[a][1]] = 0x35
    f = c.fork(a)
    assert (c.k.view(torch.uint8)[:, c._pages[f][1]] == 0x35).all() and c._pages[f][1] != c._pages[a][1]
