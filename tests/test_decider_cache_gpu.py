"""The decider over its caches: prompts in pieces, forks of a prefix, tokens one by one, against the uncached forward."""
from __future__ import annotations

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["decider", "tiny"])
def models(request):
    """(model with the kernels, its logits on the packed prompts by transformers' eager layers)."""
    from fastdecisions_amd.model import DECIDER_4_LAYERS, TINY, build_decider, install_hip_kernels, synthetic_ids
    shape = DECIDER_4_LAYERS if request.param == "decider" else TINY
    model = build_decider(shape, seed=3)
    prompts = [synthetic_ids(1, n, shape.vocab_size, seed=n) for n in (333, 97, 210)]
    with torch.no_grad():
        eager = [model(p) for p in prompts]
        install_hip_kernels(model)
        hip = [model(p) for p in prompts]
    return model, prompts, eager, hip


def spread(models):
    """How far two bf16 evaluations of the model are apart: the uncached kernels' and the eager layers'."""
    _, _, eager, hip = models
    return max(((h - e).norm() / e.norm()).item() for h, e in zip(hip, eager))


def far(a, b):
    return ((a - b).norm() / b.norm()).item()


# cut into pieces on both sides of the delta rule's change of form
CUTS = {333: [1, 64, 8, 130, 1, 1, 128], 97: [90, 7], 210: [1] * 10 + [200]}


def feed(model, cache, prompts):
    """Every prompt in its pieces, the i-th pieces of all of them in one step: letter logits per prompt."""
    slots = [cache.open() for _ in prompts]
    cuts = [CUTS[p.shape[1]] for p in prompts]
    done, out = [0] * len(prompts), [[] for _ in prompts]
    for i in range(max(map(len, cuts))):
        live = [r for r in range(len(prompts)) if i < len(cuts[r])]
        ids = torch.cat([prompts[r][:, done[r]:done[r] + cuts[r][i]] for r in live], dim=1)
        step = cache.step([slots[r] for r in live], [cuts[r][i] for r in live])
        logits = model(ids, cache=step)
        at = 0
        for r in live:
            out[r].append(logits[:, at:at + cuts[r][i]])
            at += cuts[r][i]
            done[r] += cuts[r][i]
    assert done == [p.shape[1] for p in prompts]
    return slots, [torch.cat(o, dim=1) for o in out]


@torch.no_grad()
def test_prompts_in_pieces(models):
    """The cached forward is another bf16 evaluation of the same function, with its roundings at the same places
    (the attention's and the delta rule's inside): it may be as far from the uncached kernels as those are
    from the eager layers, each measured against the other's error in two directions."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("decider in pieces")
    model, prompts, eager, hip = models
    cache = DeciderCache(model.shape, requests=3, tokens=700, page_size=16)
    _, got = feed(model, cache, prompts)
    for g, h in zip(got, hip):
        assert far(g, h) <= 2 * spread(models)


@torch.no_grad()
def test_prompts_in_pieces_over_an_8_bit_cache(models):
    """e4m3 keys and values: off by up to 2^-4 of a value, 2^-5 on average, in one layer of four.  Scores and values
    move the attention's output by less than that together, and it is a part of what the logits sum."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("decider in pieces, e4m3 cache")
    model, prompts, eager, hip = models
    cache = DeciderCache(model.shape, requests=3, tokens=700, kv_dtype=torch.float8_e4m3fn)
    slots, got = feed(model, cache, prompts)
    for g, h in zip(got, hip):
        assert far(g, h) <= 2 * spread(models) + 2.0 ** -4
    k, v = cache.read(slots[1], 3)
    assert k.shape == v.shape == (1, model.shape.num_key_value_heads, 97, model.shape.head_dim)
    assert torch.isfinite(k).all() and k.abs().amax(-1).min() > 0


@torch.no_grad()
def test_questions_over_a_shared_prefix(models):
    """Forks of a prefix, each with its own question, in one packed step: the logits of prefix + question, and
    the parent can still be continued afterwards."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("questions over a prefix")
    model, prompts, _, _ = models
    prefix, questions = prompts[0], [prompts[1][:, :30], prompts[2][:, :1], prompts[1][:, 40:97]]
    cache = DeciderCache(model.shape, requests=5, tokens=1000, page_size=32)
    parent = cache.open()
    model(prefix, cache=cache.step([parent], [333]))
    forks = [cache.fork(parent) for _ in questions]
    lens = [q.shape[1] for q in questions]
    step = cache.step(forks, lens)
    logits = model(torch.cat(questions, dim=1), cache=step)
    for r, (q, last) in enumerate(zip(questions, step.last_rows)):
        want = model(torch.cat([prefix, q], dim=1))[:, 333:]
        assert far(logits[:, last + 1 - lens[r]:last + 1], want) <= 2 * spread(models), r
    for f in forks:
        cache.close(f)
    after = model(questions[0], cache=cache.step([parent], [30]))
    want = model(torch.cat([prefix, questions[0]], dim=1))[:, 333:]
    assert far(after, want) <= 2 * spread(models)


@torch.no_grad()
def test_slot_readout_over_the_cache(models):
    """The slot-only readout on a step's last rows equals the logits there."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("slot readout over the cache")
    model, prompts, _, _ = models
    caches = [DeciderCache(model.shape, requests=2, tokens=500) for _ in range(2)]
    ids = torch.cat([prompts[1], prompts[2]], dim=1)
    steps = [c.step([c.open(), c.open()], [97, 210]) for c in caches]
    rows = torch.tensor(steps[0].last_rows, dtype=torch.int32, device="cuda")
    logits, _ = model.slot_logits(ids, torch.zeros_like(rows), rows, cache=steps[0])
    whole = model(ids, cache=steps[1])
    # logits are sums in fp32 of bf16 products, rounded to bf16: two orders of summation are one step apart
    assert (logits - whole[0, rows.long()]).abs().max() <= 2 * 2.0 ** -8 * whole.abs().max()


@torch.no_grad()
def test_tokens_from_a_replayed_graph(models):
    """One captured step of a token per request, replayed with CacheStep.again: the eager steps' logits, bit for bit."""
    from fastdecisions_amd.decider_cache import DeciderCache
    announce("captured token steps")
    model, prompts, _, _ = models
    runs = []
    for captured in (False, True):
        cache = DeciderCache(model.shape, requests=2, tokens=600, max_tokens=400, page_size=16)
        slots = [cache.open(), cache.open()]
        model(torch.cat([prompts[0], prompts[1]], dim=1), cache=cache.step(slots, [333, 97]))
        ids = prompts[2][:, :2].clone()
        out = []
        if not captured:
            for t in range(6):
                out.append(model(prompts[2][:, 2 * t:2 * t + 2], cache=cache.step(slots, [1, 1])))
        else:
            step = cache.step(slots, [1, 1])
            saved = [t.clone() for t in (cache.conv, cache.delta)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                model(ids, cache=step)                     # warm up: keys and values are rewritten below,
            torch.cuda.current_stream().wait_stream(side)
            for t, s in zip((cache.conv, cache.delta), saved):
                t.copy_(s)                                 # the states are put back
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                logits = model(ids, cache=step)
            for t in range(6):
                if t:
                    step.again()
                ids.copy_(prompts[2][:, 2 * t:2 * t + 2])
                graph.replay()
                torch.cuda.synchronize()
                out.append(logits.clone())
        runs.append(out)
    for eager, replayed in zip(*runs):
        assert torch.equal(eager, replayed)


@torch.no_grad()
def test_what_the_cached_forward_refuses(models):
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider
    model, prompts, _, _ = models
    cache = DeciderCache(model.shape, requests=1, tokens=200)
    step = cache.step([cache.open()], [10])
    with pytest.raises(ValueError, match="ids"):
        model(prompts[1], cache=step)
    plain = build_decider(TINY, seed=4)
    small = DeciderCache(TINY, requests=1, tokens=100)
    with pytest.raises(RuntimeError, match="install_hip_kernels"):
        plain(prompts[1][:, :10] % TINY.vocab_size, cache=small.step([small.open()], [10]))


@torch.no_grad()
def test_an_empty_request_reads_as_no_rows():
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY
    announce("decider cache, an empty request")
    cache = DeciderCache(TINY, requests=2, tokens=64)
    layer = next(iter(cache._attention))
    k, v = cache.read(cache.open(), layer)
    assert k.shape == v.shape == (1, TINY.num_key_value_heads, 0, TINY.head_dim)


def test_ops_trace():
    """opcheck of the cache operators' ops: schema (what they mutate), fakes, AOT dispatch."""
    import fastdecisions_amd.cached_ops as ops
    from cache_reference import make_pages
    announce("opcheck of the cache ops")
    cu = torch.tensor([0, 3, 3, 20], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 5, 17], dtype=torch.int32, device="cuda")
    idx = torch.tensor([2, 0, 4], dtype=torch.int32, device="cuda")
    r = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        for fp8 in (False, True):
            c = make_pages([40, 5, 17], 16, 4, 128, fp8, seed=1)
            k, v, q = r(1, 20, 4, 128).transpose(1, 2), r(1, 20, 4, 128).transpose(1, 2), r(1, 20, 16, 128).transpose(1, 2)
            # (test_schema and AOT dispatch do arithmetic on their inputs, which torch has not for 8-bit floats)
            tests = ("test_faketensor",) if fp8 else ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
            check = lambda op, args: torch.library.opcheck(op, args, test_utils=tests)
            check(ops.paged_gqa_op, (q, c["k"], c["v"], c["table"], lens, c["ks"], c["vs"], q.clone(), cu, 17))
            check(ops.paged_kv_read_op, (c["k"], c["v"], c["table"], cu, 20, c["ks"], c["vs"]))
            if not fp8:
                check(ops.paged_kv_write_op, (k, v, c["k"], c["v"], c["table"], lens, None, None, cu))
        check(ops.packed_conv_state_op, (r(1, 20, 6144), r(6144, 1, 4), r(6, 3, 6144), cu, idx))
        g, beta = -torch.rand((1, 20, 16), device="cuda"), torch.rand((1, 20, 16), device="cuda").to(torch.bfloat16)
        check(ops.gated_delta_step_op, (r(1, 20, 16, 128), r(1, 20, 16, 128), r(1, 20, 16, 128), g, beta,
                                        torch.randn((6, 16, 128, 128), device="cuda"), cu, idx))
