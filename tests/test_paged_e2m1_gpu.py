"""The 4-bit paged cache on the GPU: writing, reading and attention against float64 forms of their definitions."""
from __future__ import annotations

import pytest
import torch

from cache_reference import attention
from e2m1_reference import codes, hold, make_pages4, pack, rows4, values
from helpers import announce
from test_paged_cache_gpu import ints, make_q, run_attention, starts

pytestmark = pytest.mark.gpu


def check(c, q, out, lens, new, gate=None, packed=True, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    at = starts(new)
    for r, n in enumerate(new):
        take = (lambda t: t[0, :, at[r]:at[r + 1]]) if packed else (lambda t: t[r])
        k, there = rows4(c, "k", r, lens[r])
        v, _ = rows4(c, "v", r, lens[r])
        want, bound = attention(take(q), (k, v.nan_to_num(0.0), there), lens[r], scale, None if gate is None else take(gate))
        # a row is NaN where a key that it sees is (its own probability of it is never 0 here), and nowhere else
        keys = torch.arange(lens[r], device="cuda")
        seen = (keys <= (lens[r] - n + torch.arange(n, device="cuda"))[:, None]) & there
        odd = (seen.double() @ torch.isnan(v).double()).repeat_interleave(q.shape[1] // v.shape[0], 0) > 0
        want = want.masked_fill(odd, torch.nan)
        got = take(out).double()
        assert torch.isnan(got).equal(torch.isnan(want)), f"request {r}"
        off = torch.where(torch.isnan(want), 0.0, (got - want).abs() - bound)
        worst = off.max().item() if n else 0.0
        assert worst <= 0, f"request {r} of {lens[r]} keys, {n} new: off by {worst:.3g} more than its bound"


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 128), (8, 2, 256), (16, 4, 64), (3, 3, 128), (6, 1, 64), (40, 1, 128)])
def test_single_tokens(hq, hkv, dim, page):
    lens = [1, 2, 31, 32, 33, 127, 128, 129, 255, 257, 1000, 2049, 0, 4111]
    new = [1] * len(lens)
    announce(f"4-bit attention, single tokens {hq}/{hkv} x {dim}, page {page}")
    c = make_pages4(lens, page, hkv, dim, seed=dim + page)
    q = make_q(new, hq, dim, 1, packed=False)
    check(c, q, run_attention(c, q, lens, new, packed=False), lens, new, packed=False)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 4, 128, 16), (8, 2, 256, 32), (16, 4, 64, 128), (5, 5, 128, 16),
                                             (6, 1, 256, 64)])
def test_packed_suffixes(hq, hkv, dim, page, gated):
    new = [40, 1, 0, 7, 133, 300, 64]
    cached = [500, 1000, 77, 0, 1, 2500, 64]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"4-bit attention, packed suffixes {hq}/{hkv} x {dim}, page {page}, gated {gated}")
    c = make_pages4(lens, page, hkv, dim, seed=dim + page)
    q = make_q(new, hq, dim, 2)
    gate = make_q(new, hq, dim, 3) if gated else None
    check(c, q, run_attention(c, q, lens, new, gate=gate), lens, new, gate=gate)


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_each_kernel_takes_any_lengths(dim, rows):
    """max_seqlen chooses the kernel and bounds nothing: tiles of 16 rows, of 32 and of 128."""
    new, cached = [200, 1, 30, 70], [700, 900, 0, 60]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"4-bit attention x {dim}, the kernel for {rows} tokens")
    c = make_pages4(lens, 16, 2, dim, seed=5)
    q = make_q(new, 4, dim, 4)
    check(c, q, run_attention(c, q, lens, new, max_seqlen=rows), lens, new)


@pytest.mark.parametrize("new", [[3100], [1333, 1400, 1500]])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 64), (3, 1, 128), (4, 2, 256)])
def test_prompts(new, hq, hkv, dim):
    announce(f"4-bit attention, prompts {new}, {hq}/{hkv} x {dim}")
    c = make_pages4(new, 64, hkv, dim, seed=26)
    q = make_q(new, hq, dim, 27)
    check(c, q, run_attention(c, q, new, new), new, new)


@pytest.mark.parametrize("n", [1, 40])
def test_many_requests(n):
    lens = [n + (i * 37) % 300 for i in range(149)] + [6000]
    announce(f"4-bit attention, 150 requests of {n}")
    c = make_pages4(lens, 16, 2, 64, seed=6)
    q = make_q([n] * 150, 8, 64, 5, packed=False)
    check(c, q, run_attention(c, q, lens, [n] * 150, packed=False), lens, [n] * 150, packed=False)


@pytest.mark.parametrize("n", [1, 9])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 64), (16, 4, 128), (8, 2, 256)])
def test_long_caches(hq, hkv, dim, n):
    """So many keys that a wavefront takes many blocks of them, each staged where an earlier one lay."""
    lens = [4000 + 517 * i for i in range(16)] + [9] * 60 + [70000]
    announce(f"4-bit attention, long caches, {n} new, {hq}/{hkv} x {dim}")
    c = make_pages4(lens, 64, hkv, dim, seed=8)
    q = make_q([n] * len(lens), hq, dim, 9, packed=False)
    check(c, q, run_attention(c, q, lens, [n] * len(lens), packed=False), lens, [n] * len(lens), packed=False)


@pytest.mark.parametrize("n", [1, 50])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_absent_pages_and_nan_behind_the_keys(dim, n):
    """Keys on no page are not seen; blocks of NaN behind the last key, and at keys a row does not see, do not
    reach it; at keys that it sees they do."""
    lens, new = [300, 500, 64 + n, 200 + n], [n] * 4
    announce(f"4-bit attention, absent pages and NaN, {n} new x {dim}")
    c = make_pages4(lens, 16, 2, dim, seed=9)
    c["table"][0, 2:7] = -1
    c["table"][1, 0] = c["k"].shape[0] + 5
    for r, length in enumerate(lens):  # what lies behind the last key on its page
        at = length % 16
        if at:
            c["ks"][c["table"][r, length // 16], :, at:] = 255
            c["vs"][c["table"][r, length // 16], :, at:] = 255
    last = lens[3] - 1
    c["vs"][c["table"][3, last // 16], 0, last % 16, 1] = 255   # seen by the last token alone
    q = make_q(new, 8, dim, 10, packed=False)
    check(c, q, run_attention(c, q, lens, new, packed=False), lens, new, packed=False)


def test_strided_pools():
    """Heads inside and outside the page, spare rows and features between: strides of any kind."""
    lens, new = [100, 333], [1, 1]
    announce("4-bit attention, strided pools")
    for inside in (False, True):
        c = make_pages4(lens, 32, 3, 128, seed=11)
        plain = dict(c)
        for name in ("k", "v"):
            pool, scale = c[name].view(torch.uint8), c[name + "s"]
            if inside:
                w = torch.zeros((pool.shape[0], 32, 5, 80), dtype=torch.uint8, device="cuda")[:, :, 1:4, 16:]
                w.copy_(pool.transpose(1, 2))
                c[name] = w.transpose(1, 2).view(torch.float4_e2m1fn_x2)
                ws = torch.zeros((pool.shape[0], 5, 40, 4), dtype=torch.uint8, device="cuda")[:, 1:4, 4:36]
            else:
                w = torch.zeros((pool.shape[0], 4, 40, 64), dtype=torch.uint8, device="cuda")[:, 1:, 8:]
                w.copy_(pool)
                c[name] = w.view(torch.float4_e2m1fn_x2)
                ws = torch.zeros((pool.shape[0], 4, 33, 4), dtype=torch.uint8, device="cuda")[:, 1:, 1:]
            ws.copy_(scale)
            c[name + "s"] = ws
        q = make_q(new, 6, 128, 12, packed=False)
        check(plain, q, run_attention(c, q, lens, new, packed=False), lens, new, packed=False)
        q = make_q([90, 300], 6, 128, 13)
        check(plain, q, run_attention(c, q, lens, [90, 300]), lens, [90, 300])


# ---------------------------------------------------------------- writing and reading

def extremes(gen, shape):
    """Rows of every magnitude: zeros, subnormals, ties, the largest numbers, infinities, NaN."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x = (x * torch.exp2(torch.randint(-140, 120, (*shape[:-1], 1), generator=gen, device="cuda").float())).to(torch.bfloat16)
    flat = x.view(-1, shape[-1])
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -5.0, 0.0, -0.0], device="cuda")
    flat[0] = 0.0
    flat[1] = -0.0
    flat[2, :13] = ties.to(torch.bfloat16)
    flat[3, :13] = (ties * 2.0 ** 100).to(torch.bfloat16)
    flat[4, 5], flat[4, 6] = float("inf"), -float("inf")
    flat[5, 40], flat[5, 3] = float("nan"), 1.0
    flat[6, :6] = torch.tensor([3.38e38, -3.38e38, 2.9e38, 2.6e38, 2.2e38, 1e38], device="cuda").to(torch.bfloat16)
    flat[7] = float("inf")
    flat[8, 0] = 2.0 ** -133
    flat[9, :2] = torch.tensor([3.38e38, float("inf")], device="cuda").to(torch.bfloat16)
    return x


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,dim,page", [(4, 128, 16), (2, 256, 64), (3, 64, 256), (1, 128, 32)])
def test_write_and_read(heads, dim, page, packed):
    """Codes and scales of every new row, nothing else touched; read back as what they stand for."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    new = [70, 1, 0, 33, 140] if packed else [37] * 4
    cached = [500, 31, 9, 0, 16][:len(new)]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"4-bit write and read, {heads} x {dim}, page {page}, packed {packed}")
    c = make_pages4(lens, page, heads, dim, seed=20)
    c["table"][1, 0] = -1
    gen = torch.Generator(device="cuda").manual_seed(21)
    shape = (1, sum(new) + 3, heads, dim) if packed else (len(new), new[0], heads, dim)
    x = {name: extremes(gen, shape).transpose(1, 2) for name in "kv"}
    want = {name: t.view(torch.uint8).clone() for name, t in c.items() if name in ("k", "v", "ks", "vs")}
    at = starts(new)
    for name in "kv":
        for r, n in enumerate(new):
            y = x[name][0, :, at[r]:at[r + 1]] if packed else x[name][r]
            code, scale = hold(y.double())
            pos = lens[r] - n + torch.arange(n, device="cuda")
            pages = c["table"][r].long()[pos // page]
            live = pages >= 0
            byte = pack(code).view(torch.uint8).transpose(0, 1)
            want[name][pages[live], :, (pos % page)[live]] = byte[live]
            want[name + "s"][pages[live], :, (pos % page)[live]] = scale.transpose(0, 1)[live]
    cu = ints(starts(new)) if packed else None
    paged_kv_write(x["k"], x["v"], c["k"], c["v"], c["table"], ints(lens), k_scale=c["ks"], v_scale=c["vs"], cu_seqlens=cu)
    for name in "kv":
        assert torch.equal(c[name + "s"], want[name + "s"]), name
        nan = (want[name + "s"] == 255)[..., None].expand(*want[name + "s"].shape, 32).flatten(-2)
        got, expect = codes(c[name]), codes(want[name].view(torch.float4_e2m1fn_x2))
        assert torch.equal(got.masked_fill(nan, 0), expect.masked_fill(nan, 0)), name
    total = sum(lens)
    k, v = paged_kv_read(c["k"], c["v"], c["table"], ints(starts(lens)), total, k_scale=c["ks"], v_scale=c["vs"])
    for name, out in (("k", k), ("v", v)):
        assert out.shape == (1, heads, total, dim)
        for r, n in enumerate(lens):
            rows, there = rows4(c, name, r, n)
            rows = torch.where(there[None, :, None], rows, 0.0)
            got = out[0, :, starts(lens)[r]:starts(lens)[r + 1]].double()
            assert torch.equal(torch.nan_to_num(got, nan=12345.0), torch.nan_to_num(rows, nan=12345.0)), (name, r)
            assert not torch.isinf(got).any()


def test_every_code_and_scale_reads_as_its_value():
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read
    announce("4-bit read, every byte and scale")
    byte = torch.arange(256, device="cuda", dtype=torch.uint8)
    pool = byte.repeat(2)[None, None].expand(16, 16, 512).reshape(16, 1, 16, 16, 32)[:, :, :, :, :].reshape(256, 1, 16, 32)
    scale = torch.arange(256, device="cuda", dtype=torch.uint8)[:, None, None, None].expand(256, 1, 16, 2).contiguous()
    k = pool.contiguous().view(torch.float4_e2m1fn_x2)
    table = torch.arange(256, device="cuda", dtype=torch.int32)[None]
    got, _ = paged_kv_read(k, k, table, ints([0, 4096]), 4096, k_scale=scale, v_scale=scale)
    want = values(k, scale).permute(1, 0, 2, 3).reshape(1, 4096, 64)
    over = want.abs() >= 2.0 ** 128   # no bf16 number; the write makes none
    assert torch.equal(torch.isnan(got[0]), torch.isnan(want))
    fine = ~over & ~torch.isnan(want)
    assert torch.equal(got[0].double()[fine], want[fine])


def test_a_step_in_a_graph_grows():
    """Write and attend, captured once and replayed as the request grows, each replay against an eager step."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_write
    announce("4-bit write and attention in a graph")
    lens = [200, 1500]
    c = make_pages4([n + 8 for n in lens], 64, 2, 128, seed=30)
    gen = torch.Generator(device="cuda").manual_seed(31)
    x = [torch.randn((2, 1, h, 128), generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2) for h in (8, 2, 2)]
    q, k, v = (t.clone() for t in x)
    at = ints(lens)

    def step(c, q, k, v, at):
        from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
        paged_kv_write(k, v, c["k"], c["v"], c["table"], at, k_scale=c["ks"], v_scale=c["vs"])
        return paged_gqa_attention(q, c["k"], c["v"], c["table"], at, k_scale=c["ks"], v_scale=c["vs"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c, q, k, v, at)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c, q, k, v, at)
    # the run before the capture has written a key
    eager = {k: (v.clone() if torch.is_tensor(v) and k != "table" else v) for k, v in c.items()}
    for i in range(4):
        now = [torch.randn(t.shape, generator=gen, device="cuda").to(torch.bfloat16) for t in (q, k, v)]
        at.copy_(ints([n + 1 + i for n in lens]))
        for held, t in zip((q, k, v), now):
            held.copy_(t)
        graph.replay()
        want = step(eager, *now, ints([n + 1 + i for n in lens]))
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
