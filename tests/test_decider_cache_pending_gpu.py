"""Evictions of requests with a step that has not run, over the model."""
from __future__ import annotations

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu


@torch.no_grad()
def test_a_step_that_has_not_run_holds_back_an_eviction():
    """Refused before anything moves; run or taken back, the request goes on as one that nobody tried to cut."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce("an eviction before a step has run")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 80, TINY.vocab_size, seed=1)
    out = []
    for refused in (False, True):
        cache = DeciderCache(TINY, requests=1, tokens=100, page_size=16, key_weights=True)
        a = cache.open()
        model(ids[:, :40], cache=cache.step([a], [40]))
        if refused:
            step = cache.step([a], [10])
            with pytest.raises(RuntimeError, match="has not run"):
                cache.evict([a], 20)
            step.cancel()
            assert (cache.length(a), cache.position(a)) == (40, 40)
        step = cache.step([a], [10])
        if refused:
            with pytest.raises(RuntimeError, match="has not run"):
                cache.evict([a], 20)
        got = [model(ids[:, 40:50], cache=step)]
        cache.evict([a], 20, recent=4)
        assert (cache.length(a), cache.position(a)) == (20, 50)
        step = cache.step([a], [1])
        got.append(model(ids[:, 50:51], cache=step))
        if refused:
            step.again()
            with pytest.raises(RuntimeError, match="has not run"):
                cache.evict([a], 12)
            step.cancel()
        got += [cache.weights.clone(), *cache.read(a, 3)]
        out.append(got)
    assert all(torch.equal(x, y) for x, y in zip(*out))


@torch.no_grad()
def test_recorded_steps_and_single_layers_hold_back_nothing():
    """A graph's replays are not seen, and neither are layers called by themselves, but the layers' own sign."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce("evictions behind replays and single layers")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 41, TINY.vocab_size, seed=1)
    cache = DeciderCache(TINY, requests=2, tokens=200, page_size=16, key_weights=True)
    a, b = cache.open(), cache.open()
    model(ids[:, :40], cache=cache.step([a], [40]))
    step, new = cache.step([a], [1]), ids[:, 40:].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model(new, cache=step)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model(new, cache=step)
    step.again()
    graph.replay()
    torch.cuda.synchronize()
    cache.evict([a], 16)
    assert (cache.length(a), cache.position(a)) == (16, 42)
    step = cache.step([b], [30])
    layer = model.core.layers[3].self_attn
    x = torch.randn((1, 30, TINY.hidden_size), device="cuda").to(torch.bfloat16)
    layer(x, model.core.rotary_emb(x, step.positions), fd_cache=step)
    cache.evict([b], 16)
    assert cache.length(b) == 16 and torch.isfinite(cache.read(b, 3)[0]).all()
