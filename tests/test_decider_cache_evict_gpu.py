"""The decider over 4-bit caches and over requests that were cut to the keys that mattered."""
from __future__ import annotations

import pytest
import torch

from helpers import announce
from test_decider_cache_gpu import far, feed, models, spread  # noqa: F401  (models: the fixture)
from test_evict_gpu import chosen

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2]


@torch.no_grad()
def test_prompts_in_pieces_over_a_4_bit_cache(models):  # noqa: F811
    """e2m1 keys and values: off by up to 2^-2 of a value (half a step of one mantissa bit), in one layer of four; as for
    the 8-bit cache, whose half step is 2^-4, scores and values move the attention's output by less than that together."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("decider in pieces, 4-bit cache")
    model, prompts, eager, hip = models
    cache = DeciderCache(model.shape, requests=3, tokens=700, kv_dtype=torch.float4_e2m1fn_x2)
    slots, got = feed(model, cache, prompts)
    for g, h in zip(got, hip):
        assert far(g, h) <= 2 * spread(models) + 2.0 ** -2
    k, v = cache.read(slots[1], 3)
    assert k.shape == v.shape == (1, model.shape.num_key_value_heads, 97, model.shape.head_dim)
    assert torch.isfinite(k).all() and k.abs().amax(-1).min() > 0


@torch.no_grad()
@pytest.mark.parametrize("observe", [None, 16])
def test_weights_that_the_keys_have_drawn(models, observe):  # noqa: F811
    """Every counted token gives each key head its group's probabilities, which sum to 1 per query head; the first key
    draws from every token, the last one from itself alone; and the logits are those without weights, bit for bit."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce(f"decider, key weights, observe {observe}")
    model, prompts, _, _ = models
    shape = model.shape
    plain = DeciderCache(shape, requests=2, tokens=700, page_size=16)
    cache = DeciderCache(shape, requests=2, tokens=700, page_size=16, key_weights=True, observe=observe)
    counted = {}
    for c in (plain, cache):
        c.out, slots = [], [c.open(), c.open()]
        for ids, lens in ((torch.cat([prompts[0][:, :300], prompts[1]], 1), [300, 97]), (prompts[2][:, :2], [1, 1])):
            c.out.append(model(ids, cache=c.step(slots, lens)))
            for s, n in zip(slots, lens):
                counted[s] = counted.get(s, 0) * (c is cache) * (len(c.out) > 1) + min(n, observe or n)
    assert all(torch.equal(a, b) for a, b in zip(plain.out, cache.out))
    group = shape.num_attention_heads // shape.num_key_value_heads
    layer = next(iter(cache._attention))
    w = cache.key_weights(layer)
    for s, length in zip(slots, (301, 98)):
        total = w[s].double().sum(-1)
        # a row's probabilities sum to 1 up to the fp32 roundings of its denominator and of each of them
        assert ((total - counted[s] * group).abs() <= 1e-4 * counted[s] * group).all()
        assert (w[s, :, length:] == 0).all() and (w[s, :, :length] > 0).all()


@torch.no_grad()
@pytest.mark.parametrize("kv_dtype", KINDS)
def test_a_prefix_cut_and_forked(models, kv_dtype):  # noqa: F811
    """Weights, eviction, fork and continuation together: the kept rows are those of largest weight, and a question over
    the cut prefix is answered as over the whole one without the evicted keys (a page of them here, hidden from an uncut
    request's step): the same keys in another split, so as near as two evaluations of the model are."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce(f"decider, a prefix cut and forked, {kv_dtype}")
    model, prompts, _, _ = models
    layer = 3
    prefix, question = prompts[0], prompts[1][:, :30]
    caches = [DeciderCache(model.shape, requests=3, tokens=1200, page_size=16, key_weights=True, kv_dtype=kv_dtype) for _ in range(2)]
    slots = [c.open() for c in caches]
    for c, s in zip(caches, slots):
        model(prefix, cache=c.step([s], [333]))
    cut, whole = caches
    # by weight: 100 keys, the last 20 among them
    f = cut.fork(slots[0])
    k, v = cut.read(f, layer)
    w = cut.key_weights(layer)[f].clone()
    cut.evict([f], 100, recent=20)
    k2, v2 = cut.read(f, layer)
    for h in range(w.shape[0]):
        mine = torch.tensor(chosen(w[h].tolist(), 333, 100, 20), device="cuda")
        assert torch.equal(k2[0, h], k[0, h, mine]) and torch.equal(v2[0, h], v[0, h, mine])
        assert torch.equal(cut.key_weights(layer)[f, h, :100], w[h, mine]) and (cut.key_weights(layer)[f, h, 100:] == 0).all()
    assert cut.position(f) == 333
    logits = model(question, cache=cut.step([f], [30]))
    assert torch.isfinite(logits).all()
    # the same as hiding the evicted keys
    cut.weights[:, slots[0], :, 32:48] = -1.0
    cut.evict([slots[0]], 333 - 16)
    got = model(question, cache=cut.step([slots[0]], [30]))
    step = whole.step([slots[1]], [30])
    step.page_table[0, 2] = -1
    want = model(question, cache=step)
    assert far(got, want) <= 2 * spread(models)
    # and the parent's other fork still has what it shared
    g = cut.fork(f)
    assert cut.length(g) == 130 and cut.position(g) == 363


@torch.no_grad()
def test_captured_steps_gather_weights(models):  # noqa: F811
    """A step of tokens with weights, captured and replayed: the eager steps' sums, bit for bit."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("decider, captured steps with key weights")
    model, prompts, _, _ = models
    runs = []
    for captured in (False, True):
        cache = DeciderCache(model.shape, requests=2, tokens=600, max_tokens=400, page_size=16, key_weights=True,
                             kv_dtype=torch.float4_e2m1fn_x2)
        slots = [cache.open(), cache.open()]
        model(torch.cat([prompts[0], prompts[1]], dim=1), cache=cache.step(slots, [333, 97]))
        ids = prompts[2][:, :2].clone()
        if not captured:
            for t in range(4):
                model(prompts[2][:, 2 * t:2 * t + 2], cache=cache.step(slots, [1, 1]))
        else:
            step = cache.step(slots, [1, 1])
            saved = [t.clone() for t in (cache.conv, cache.delta, cache.weights)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                model(ids, cache=step)
            torch.cuda.current_stream().wait_stream(side)
            for t, s in zip((cache.conv, cache.delta, cache.weights), saved):
                t.copy_(s)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                model(ids, cache=step)
            for t in range(4):
                if t:
                    step.again()
                ids.copy_(prompts[2][:, 2 * t:2 * t + 2])
                graph.replay()
                torch.cuda.synchronize()
        runs.append(cache.weights.clone())
    assert torch.equal(*runs)


def test_ops_trace():
    """opcheck of the ops: schema (what they mutate), fakes, AOT dispatch."""
    import fastdecisions_amd.cached_ops as ops
    from cache_reference import make_pages
    from e2m1_reference import make_pages4
    announce("opcheck of the weights' and the eviction's ops")
    cu = torch.tensor([0, 3, 3, 20], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 5, 17], dtype=torch.int32, device="cuda")
    idx = torch.tensor([2, 0, 3], dtype=torch.int32, device="cuda")
    r = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        for c in (make_pages([40, 5, 17], 16, 4, 128, False, seed=1), make_pages4([40, 5, 17], 16, 4, 128, seed=1)):
            w = torch.rand((4, 4, c["table"].shape[1] * 16), device="cuda")
            new = torch.arange(3, dtype=torch.int32, device="cuda")[:, None] + c["k"].shape[0] - 3  # nobody's
            # (test_schema and AOT dispatch do arithmetic on their inputs, which torch has not for 4-bit floats)
            tests = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic") if c["ks"] is None else ("test_faketensor",)
            check = lambda op, args: torch.library.opcheck(op, args, test_utils=tests)
            check(ops.paged_key_weights_op, (r(1, 20, 16, 128).transpose(1, 2), c["k"], c["table"], lens, w, c["ks"], cu, 17, 5, idx))
            check(ops.paged_kv_evict_op, (c["k"], c["v"], c["table"], lens, w, new, 16, 4, c["ks"], c["vs"], idx))
            if c["ks"] is not None:
                check(ops.paged_kv_read_op, (c["k"], c["v"], c["table"], cu, 20, c["ks"], c["vs"]))
