"""Cached forwards under torch.compile's tracing, and the op of the chunked delta rule between states."""
from __future__ import annotations

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("new", [2, 40])
def test_a_cached_step_traces_whole(new):
    """A token step and a prompt piece (the two forms of the delta rule) are graphs without a break; the traced
    calls are the eager ones, bit for bit."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce(f"traced cached step of {new} tokens")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 2 * new, TINY.vocab_size, seed=1)
    torch._dynamo.reset()
    traced = torch.compile(lambda i, step: model(i, cache=step), backend="eager", fullgraph=True)
    out = []
    for call in (lambda i, step: model(i, cache=step), traced):
        cache = DeciderCache(TINY, requests=1, tokens=200)
        slot = cache.open()
        out.append([call(part, cache.step([slot], [new])) for part in (ids[:, :new], ids[:, new:])])
    for eager, got in zip(*out):
        assert torch.equal(eager, got)


@torch.no_grad()
def test_the_op_of_the_rule_between_states():
    import fastdecisions_amd.cached_ops as ops
    announce("opcheck of gated_delta_rule_states")
    r = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 3, 3, 70], dtype=torch.int32, device="cuda")
    g, beta = -torch.rand((1, 70, 16), device="cuda"), torch.rand((1, 70, 16), device="cuda").to(torch.bfloat16)
    torch.library.opcheck(ops.gated_delta_rule_states_op,
                          (r(1, 70, 16, 128), r(1, 70, 16, 128), r(1, 70, 16, 128), g, beta,
                           torch.randn((3, 16, 128, 128), device="cuda"), cu),
                          test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


@torch.no_grad()
def test_refused_and_failed_forwards(monkeypatch):
    """A refused step runs afterwards as if nothing had been; after one that failed on the way its request can
    only be closed, and the others go on."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce("refused and failed cached forwards")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 60, TINY.vocab_size, seed=1)
    caches = [DeciderCache(TINY, requests=2, tokens=200) for _ in range(2)]
    slots = [[c.open(), c.open()] for c in caches]
    for c, s in zip(caches, slots):
        model(ids[:, :40], cache=c.step(s, [30, 10]))
    clean, c = caches
    want = model(ids[:, 40:50], cache=clean.step(slots[0][:1], [10]))
    step = c.step(slots[1][:1], [10])
    with pytest.raises(ValueError, match="ids"):
        model(ids[:, 40:51], cache=step)
    assert torch.equal(model(ids[:, 40:50], cache=step), want) and not c._waiting
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no gradients"):
        model(ids[:, 50:51], cache=c.step(slots[1][:1], [1]))
    c._waiting[slots[1][0]][0].cancel()

    def broken(*args, **kwargs):
        raise RuntimeError("out of memory, say")
    with monkeypatch.context() as m:
        m.setattr(model.core.layers[2].mlp, "forward", broken)
        with pytest.raises(RuntimeError, match="say"):
            model(ids[:, 50:55], cache=c.step(slots[1][:1], [5]))
    with pytest.raises(RuntimeError, match="only be closed"):
        c.step(slots[1][:1], [1])
    c.close(slots[1][0])
    want = model(ids[:, 50:53], cache=clean.step(slots[0][1:], [3]))
    assert torch.equal(model(ids[:, 50:53], cache=c.step(slots[1][1:], [3])), want)
    fresh = model(ids[:, :7], cache=c.step([c.open()], [7]))
    clean.close(slots[0][0])
    assert torch.equal(fresh, model(ids[:, :7], cache=clean.step([clean.open()], [7])))


def test_a_cache_stays_on_its_device():
    """Made on the current device, its later steps go there whichever device is current then."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY
    cache = DeciderCache(TINY, requests=1, tokens=64)
    assert cache.device == cache.k.device and cache.device.index is not None
    assert cache.step([cache.open()], [3]).buffer.device == cache.k.device


@torch.no_grad()
def test_two_streams_in_order():
    """A request closed behind a queued forward on one stream, its pages taken by another one on a second stream
    that waits for the first: both as on one stream."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce("one cache, two streams")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 90, TINY.vocab_size, seed=1)
    runs = []
    for streams in ([torch.cuda.current_stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        cache = DeciderCache(TINY, requests=1, tokens=50, page_size=16)
        out, last = [], torch.cuda.current_stream()
        for i in range(6):
            stream = streams[i % 2]
            stream.wait_stream(last)
            with torch.cuda.stream(stream):
                slot = cache.open()
                for part in ((0, 40), (40, 41)):
                    n = part[1] - part[0]
                    out.append(model(ids[:, i + part[0]:i + part[1]], cache=cache.step([slot], [n])))
                cache.close(slot)
            last = stream
        torch.cuda.synchronize()
        runs.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
