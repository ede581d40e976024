"""Cached forwards that gather key weights under torch.compile's tracing, over pages of every type."""
from __future__ import annotations

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("kv_dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
@pytest.mark.parametrize("new", [2, 40])
def test_a_step_with_key_weights_traces_whole(kv_dtype, new, backend):
    """Without a break, also where what an op updates in place is declared to a functional graph; logits, pages, scales
    and weights are those of the eager calls, bit for bit, and an eviction afterwards finds that the steps have run."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce(f"traced step of {new} tokens with key weights, {kv_dtype}, {backend}")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 2 * new, TINY.vocab_size, seed=1)
    torch._dynamo.reset()
    traced = torch.compile(lambda i, step: model(i, cache=step), backend=backend, fullgraph=True)
    out = []
    for call in (lambda i, step: model(i, cache=step), traced):
        cache = DeciderCache(TINY, requests=1, tokens=200, kv_dtype=kv_dtype, key_weights=True, observe=16)
        slot = cache.open()
        step = cache.step([slot], [new])
        got = [call(ids[:, :new], step)]
        step = cache.step([slot], [new])
        got.append(call(ids[:, new:], step))
        got += [t.view(torch.uint8) for t in (cache.k, cache.v)] + [t for t in (cache.k_scale, cache.v_scale) if t is not None]
        got.append(cache.weights.clone())
        cache.evict([slot], new)
        out.append(got + [cache.weights, *cache.read(slot, 3)])
    for eager, got in zip(*out):
        assert torch.equal(eager, got)
