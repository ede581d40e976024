"""Attention weight per cached key on the GPU against its definition in float64."""
from __future__ import annotations

import math

import pytest
import torch

from cache_reference import make_pages, rows
from e2m1_reference import make_pages4, rows4
from helpers import announce
from test_paged_cache_gpu import ints, make_q, starts

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "e4m3", "e2m1"]
# fp32 throughout.  Per probability, relative: a score's sum of up to 256 exact products in fp32 (256 half steps of
# sum |q k|, up to 60 in log2 units here: the absolute error of the exponent, times ln 2), the exponent's own rounding
# (two, of up to 60), exp2 and the division (a few half steps); then sums of up to 2^14 positive numbers in tiles
# of 16 to 32 and the tiles in turn.  Sums of roundings in their worst case would be larger; what is added is random
# in sign, so a few standard deviations are taken: 2^-24 * (60 * sqrt(256) + 2 * 60 + sqrt(2^14)) < 2^-24 * 1300.
RELATIVE = 2.0 ** -24 * 1300


def make(held, lens, page, heads, dim, seed):
    if held == "e2m1":
        return make_pages4(lens, page, heads, dim, seed), rows4
    return make_pages(lens, page, heads, dim, held == "e4m3", seed), rows


def want_weights(c, get, q, w, lens, new, index, last=None, packed=True, scale=None):
    """float64 sums on top of w [rows, heads, width]."""
    w = w.double().clone()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    at = starts(new)
    for r, n in enumerate(new):
        length = lens[r]
        if not 0 <= index[r] < w.shape[0] or index[r] in index[:r] or n == 0 or length == 0:
            continue
        x = (q[0, :, at[r]:at[r + 1]] if packed else q[r]).double()
        k, there = get(c, "k", r, length)
        group = x.shape[0] // k.shape[0]
        pos = length - n + torch.arange(n, device="cuda")
        seen = (torch.arange(length, device="cuda") <= pos[:, None]) & there
        for h in range(x.shape[0]):
            s = torch.where(seen, (x[h] @ k[h // group].T) * scale, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            w[index[r], h // group, :length] += p[max(0, n - (last or n)):].sum(0)
    return w


def check(held, new, cached, hq, hkv, dim, page, seed, *, packed=True, last=None, index=None, absent=(), max_seqlen=None,
          scale=None):
    from fastdecisions_amd.paged_evict_kernel import paged_key_weights
    lens = [a + b for a, b in zip(cached, new)]
    c, get = make(held, lens, page, hkv, dim, seed)
    for r, at in absent:
        c["table"][r, at] = -1
    q = make_q(new, hq, dim, seed + 1, packed=packed)
    width = c["table"].shape[1] * page
    gen = torch.Generator(device="cuda").manual_seed(seed + 2)
    w = torch.rand((len(new) + 2, hkv, width + 5), generator=gen, device="cuda") * 1e-3
    index = list(range(len(new))) if index is None else index
    want = want_weights(c, get, q, w, lens, new, index, last, packed, scale)
    kw = dict(cu_seqlens=ints(starts(new)), max_seqlen=max(new) if max_seqlen is None else max_seqlen) if packed else {}
    got = w.clone()
    paged_key_weights(q, c["k"], c["table"], ints(lens), got, k_scale=c["ks"], last=last, row_indices=ints(index), scale=scale, **kw)
    again = w.clone()
    paged_key_weights(q, c["k"], c["table"], ints(lens), again, k_scale=c["ks"], last=last, row_indices=ints(index), scale=scale, **kw)
    assert torch.equal(got, again)          # nothing is added in an order of its own
    same = want == w.double()
    assert torch.equal(got[same], w[same])  # what no token sees keeps its weight
    off = ((got.double() - want).abs() / want).max().item()
    assert off <= RELATIVE, f"off by {off:.3g} relative"


@pytest.mark.parametrize("held", FORMATS)
@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 4, 128, 16), (8, 2, 256, 64), (16, 4, 64, 256), (3, 3, 128, 16),
                                             (40, 1, 64, 32)])
def test_single_tokens(hq, hkv, dim, page, held):
    lens = [1, 2, 31, 32, 33, 127, 128, 129, 255, 257, 1000, 2049, 0, 4111]
    announce(f"key weights, single tokens {hq}/{hkv} x {dim}, page {page}, {held}")
    check(held, [1] * len(lens), [n - 1 for n in lens], hq, hkv, dim, page, dim + page, packed=False)


@pytest.mark.parametrize("held", FORMATS)
@pytest.mark.parametrize("last", [None, 1, 33])
@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 4, 128, 16), (8, 2, 256, 32), (6, 1, 64, 128), (5, 5, 128, 16)])
def test_packed_suffixes(hq, hkv, dim, page, last, held):
    announce(f"key weights, packed suffixes {hq}/{hkv} x {dim}, page {page}, last {last}, {held}")
    check(held, [40, 1, 0, 7, 133, 300, 64], [500, 1000, 77, 0, 1, 2500, 64], hq, hkv, dim, page, dim, last=last)


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_either_kernel_takes_any_lengths(dim, rows):
    announce(f"key weights x {dim}, the kernels for {rows} tokens")
    check("bf16", [300, 1, 30, 70], [700, 900, 0, 60], 4, 2, dim, 16, 5, max_seqlen=rows)


@pytest.mark.parametrize("new", [[3100], [1333, 1400, 1500]])
def test_prompts(new):
    announce(f"key weights, prompts {new}")
    check("e4m3", new, [0] * len(new), 16, 4, 128, 64, 26)


@pytest.mark.parametrize("n", [1, 40])
def test_many_requests(n):
    announce(f"key weights, 150 requests of {n}")
    check("e2m1", [n] * 150, [(i * 37) % 300 for i in range(149)] + [6000], 8, 2, 64, 16, 6, packed=False)


@pytest.mark.parametrize("n", [1, 50])
def test_absent_pages(n):
    announce(f"key weights, absent pages, {n} new")
    check("bf16", [n] * 3, [300, 500, 16], 8, 2, 128, 16, 7, packed=False, absent=[(0, 2), (0, 3), (1, 0), (2, 0), (2, 1)])


@pytest.mark.parametrize("n", [1, 50])
def test_rows_of_the_pool(n):
    """Rows in any order; one named twice is the first request's, one outside the pool nobody's."""
    announce(f"key weights, row indices, {n} new")
    check("e2m1", [n] * 5, [100, 200, 30, 4, 77], 8, 2, 64, 16, 8, packed=False, index=[4, 2, 4, -1, 7])


def test_far_scores():
    """Scores of some hundreds: probabilities that are one or nothing."""
    announce("key weights, scale 4")
    from fastdecisions_amd.paged_evict_kernel import paged_key_weights
    c, get = make("bf16", [900], 16, 2, 64, 9)
    q = make_q([20], 8, 64, 10)
    w = torch.zeros((1, 2, c["table"].shape[1] * 16), device="cuda")
    want = want_weights(c, get, q, w, [900], [20], [0], scale=4.0)
    paged_key_weights(q, c["k"], c["table"], ints([900]), w, cu_seqlens=ints([0, 20]), scale=4.0)
    # scores up to about 400: the exponent is off by up to 2^-24 * 400 * (sqrt(64) + 2)
    assert ((w.double() - want).abs() <= 2.0 ** -24 * 4000 * want + 1e-30).all()
    assert torch.isfinite(w).all() and abs(w.sum().item() - 20 * 8) < 0.01


@pytest.mark.parametrize("n", [1, 6, 40])
def test_fewer_keys_than_tokens(n):
    """Requests whose lengths say that some of their tokens see nothing, or that they hold nothing."""
    announce(f"key weights, fewer keys than tokens, {n} new")
    check("bf16", [n] * 5, [-n, -n + 1, -(n // 2), 3, 700], 8, 2, 64, 16, 11, packed=False)


def test_thousands_of_requests():
    """More row tiles than any number of rounds: no request is cut, and all are whole."""
    announce("key weights, 2300 requests")
    check("e2m1", [1] * 2300, [(i * 37) % 90 for i in range(2300)], 4, 4, 64, 16, 12, packed=False)
    check("bf16", [20] * 700, [(i * 37) % 90 for i in range(700)], 4, 4, 64, 16, 13, packed=False)


@pytest.mark.parametrize("n", [1, 4, 90])
def test_a_key_that_is_nan(n):
    """The rows that see it are NaN and with them the weights of every key that they see; no other key's."""
    from fastdecisions_amd.paged_evict_kernel import paged_key_weights
    announce(f"key weights, a key that is NaN, {n} new")
    length = 300 + n
    c, get = make("bf16", [length], 16, 2, 64, 14)
    q = make_q([n], 4, 64, 15)
    w = torch.zeros((1, 2, c["table"].shape[1] * 16), device="cuda")
    for key, first in ((100, 0), (300 + n // 2, n // 2)):  # seen by all tokens, by the later half
        k, got = c["k"].clone(), w.clone()
        k[c["table"][0, key // 16].long(), 1, key % 16, 5] = float("nan")
        paged_key_weights(q, k, c["table"], ints([length]), got, cu_seqlens=ints([0, n]))
        assert torch.isfinite(got[0, 0]).all()
        assert torch.isnan(got[0, 1, :length]).all()      # the last token sees them all
        last = torch.full((1, 2, w.shape[2]), 0.0, device="cuda")
        before = n // 2
        if first and before:
            paged_key_weights(q[:, :, :before], k, c["table"], ints([300 + before]), last, cu_seqlens=ints([0, before]))
            assert torch.isfinite(last).all()
    # a token that is NaN itself weighs the keys up to its own, and none behind it
    if n > 1:
        odd, got = q.clone(), w.clone()
        odd[0, 1, n // 2, 3] = float("nan")               # a query head of key head 0
        paged_key_weights(odd, c["k"], c["table"], ints([length]), got, cu_seqlens=ints([0, n]))
        assert torch.isfinite(got[0, 1]).all()
        assert torch.isnan(got[0, 0, :300 + n // 2 + 1]).all() and torch.isfinite(got[0, 0, 300 + n // 2 + 1:]).all()


def test_in_a_graph_as_requests_grow():
    """Weights and eviction captured once and replayed with other lengths, weights and tables: the eager results."""
    from fastdecisions_amd.paged_evict_kernel import paged_key_weights, paged_kv_evict
    announce("key weights and eviction in a graph")
    for n, held in ((1, "e2m1"), (60, "bf16")):
        c, _ = make(held, [900, 700, 160], 16, 2, 64, 16)  # the last one's pages become the new ones
        table, new_table = c["table"][:2].contiguous(), c["table"][2, :10].reshape(2, 5).contiguous()
        q = make_q([n] * 2, 8, 64, 17, packed=False)
        lens = ints([500, 300])
        w, out = (torch.zeros((2, 2, table.shape[1] * 16), device="cuda") for _ in range(2))

        def step(lens, w, out):
            paged_key_weights(q, c["k"], table, lens, w, k_scale=c["ks"])
            return paged_kv_evict(c["k"], c["v"], table, lens, w, new_table, 70, recent=9, k_scale=c["ks"], v_scale=c["vs"],
                                  weights_out=out)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(lens, w, out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept, left = step(lens, w, out)
        for i in range(4):
            lens.copy_(ints([500 + 100 * i, 60 + 200 * i]))
            w.zero_()
            out.zero_()
            graph.replay()
            got = [t.clone() for t in (kept, left, w, out)] + [c[x].view(torch.uint8).clone() for x in "kv"]
            w2, out2 = torch.zeros_like(w), torch.zeros_like(out)
            want = [*step(lens, w2, out2), w2, out2] + [c[x].view(torch.uint8) for x in "kv"]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (n, i)


@pytest.mark.parametrize("n", [1, 2, 77])
@pytest.mark.parametrize("hq,hkv", [(14, 2), (10, 2), (129, 1), (2048, 1)])
def test_groups_that_divide_no_tile(hq, hkv, n):
    announce(f"key weights, {hq}/{hkv} heads, {n} new")
    check("bf16", [n] * 2, [300, 1000 - n], hq, hkv, 64, 16, 18, packed=False, last=40)


def test_two_streams_at_once():
    """Calls side by side on streams of their own, weights of other strides: each as it is alone."""
    from fastdecisions_amd.paged_evict_kernel import paged_key_weights, paged_kv_evict
    announce("key weights and eviction on two streams")
    jobs = []
    for i, (held, n) in enumerate((("e2m1", 1), ("bf16", 130))):
        c, _ = make(held, [2100, 1800, 160], 16, 2, 64, 20 + i)
        table, new_table = c["table"][:2].contiguous(), c["table"][2, :10].reshape(2, 5).contiguous()
        q, lens = make_q([n] * 2, 8, 64, 30 + i, packed=False), ints([2100, 1800])
        store = lambda: torch.zeros((2, 2, 2200), device="cuda").transpose(0, 1)  # heads in front

        def run(w, out, c=c, table=table, new_table=new_table, q=q, lens=lens):
            paged_key_weights(q, c["k"], table, lens, w, k_scale=c["ks"])
            return *paged_kv_evict(c["k"], c["v"], table, lens, w, new_table, 80, recent=9, k_scale=c["ks"], v_scale=c["vs"],
                                   weights_out=out), w, out, c["k"].view(torch.uint8), c["v"].view(torch.uint8)
        jobs.append((run, store))
    want = [[t.clone() for t in run(store(), store())] for run, store in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    made = [(store(), store()) for _, store in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got.clear()
        for (run, _), stream, (w, out) in zip(jobs, streams, made):
            with torch.cuda.stream(stream):
                w.zero_(), out.zero_()
                got.append(run(w, out))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
