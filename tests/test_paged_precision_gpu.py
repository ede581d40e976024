"""Probabilities of the paged attention for few rows: nothing but the output is rounded."""
from __future__ import annotations

import pytest
import torch

from cache_reference import HALF_STEP, attention, make_pages, rows
from helpers import announce
from test_paged_cache_gpu import make_q, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,cached", [([1, 1, 1], [0, 190, 5000]), ([3, 8, 1], [700, 33, 2000]), ([16, 9], [900, 60])])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 128), (8, 2, 256), (16, 4, 64)])
def test_probabilities_keep_their_bits(hq, hkv, dim, new, cached, fp8):
    """Bound: a probability in two bf16 parts is off by 2^-16 of it, and 2^-12 of sum p |v| covers the fp32 scores (off by
    less than 2^-14 each), exp2 and sums; then the output's rounding, half a step of what was rounded.  Probabilities in
    one bf16 would be off by up to 2^-8 each."""
    announce(f"paged attention, precision, {new} tokens x {hq}/{hkv} x {dim}, fp8 {fp8}")
    lens = [n + c for n, c in zip(new, cached)]
    c = make_pages(lens, 16, hkv, dim, fp8, seed=40)
    q, gate = make_q(new, hq, dim, 41), make_q(new, hq, dim, 42)
    out = run_attention(c, q, lens, new, gate=gate)
    at = 0
    for r, n in enumerate(new):
        k, there = rows(c, "k", r, lens[r])
        v, _ = rows(c, "v", r, lens[r])
        take = lambda t: t[0, :, at:at + n]
        want, _ = attention(take(q), (k, v, there), lens[r], dim ** -0.5, take(gate))
        mag, _ = attention(take(q), (k, v.abs(), there), lens[r], dim ** -0.5, take(gate))
        inner = (2.0 ** -16 + 2.0 ** -12) * mag
        worst = ((take(out).double() - want).abs() - inner - HALF_STEP * (want.abs() + inner)).max().item()
        assert worst <= 0, f"request {r}: off by {worst:.3g} more than its bound"
        at += n


@pytest.mark.parametrize("n", [1, 12, 100])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_an_infinity_that_every_row_sees(dim, n):
    """In tiles without masks: its feature is that infinity, whatever the probability's parts, and the others are as they
    were."""
    announce(f"paged attention, an infinity seen by all, {n} tokens x {dim}")
    lens = [n + 1000]
    c = make_pages(lens, 16, 2, dim, False, seed=43)
    q = make_q([n], 8, dim, 44, packed=False, std=0.2)
    clean = run_attention(c, q, lens, [n], packed=False)
    for key, d, value in ((3, 1, "inf"), (500, dim - 1, "-inf"), (901, 40, "inf")):
        c["v"][c["table"][0, key // 16], :, key % 16, d] = float(value)
    out = run_attention(c, q, lens, [n], packed=False)
    for d, value in ((1, "inf"), (dim - 1, "-inf"), (40, "inf")):
        assert (out[..., d] == float(value)).all(), d
        out[..., d] = clean[..., d]
    assert torch.equal(out, clean)


def test_a_probability_of_one_times_infinity():
    """A row's largest probability is one exactly; its second part is not zero."""
    announce("paged attention, probability one")
    c = make_pages([1], 16, 1, 64, False, seed=45)
    c["v"][c["table"][0, 0], 0, 0, 9] = -float("inf")
    out = run_attention(c, make_q([1], 4, 64, 46, packed=False), [1], [1], packed=False)
    assert (out[..., 9] == -float("inf")).all() and torch.isfinite(out[..., :9]).all() and torch.isfinite(out[..., 10:]).all()
