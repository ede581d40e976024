"""Paged cache: writing, reading and attention on the GPU against float64 forms of their definitions."""
from __future__ import annotations

import pytest
import torch

from cache_reference import attention, e4m3, make_pages, pow2, rows
from helpers import announce

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def scales(c):
    return dict(k_scale=c["ks"], v_scale=c["vs"])


def run_attention(c, q, lens, new, gate=None, packed=True, **kw):
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    if packed:
        kw = dict(cu_seqlens=ints(starts(new)), max_seqlen=max(new)) | kw
    return paged_gqa_attention(q, c["k"], c["v"], c["table"], ints(lens), gate=gate, **scales(c), **kw)


def check_attention(c, q, out, lens, new, gate=None, packed=True, scale=None):
    dim = q.shape[-1]
    scale = dim ** -0.5 if scale is None else scale
    at = starts(new)
    for r, n in enumerate(new):
        take = (lambda t: t[0, :, at[r]:at[r + 1]]) if packed else (lambda t: t[r])
        k, there = rows(c, "k", r, lens[r])
        v, _ = rows(c, "v", r, lens[r])
        want, bound = attention(take(q), (k, v, there), lens[r], scale, None if gate is None else take(gate))
        got = take(out).double()
        assert torch.isfinite(got).all() or not torch.isfinite(want).all(), f"request {r}"
        worst = ((got - want).abs() - bound).max().item() if n else 0.0
        assert worst <= 0, f"request {r} of {lens[r]} keys, {n} new: off by {worst:.3g} more than its bound"


def make_q(new, hq, dim, seed, packed=True, std=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (1, sum(new), hq, dim) if packed else (len(new), new[0], hq, dim)
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(torch.bfloat16).transpose(1, 2)


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 128), (8, 2, 256), (16, 4, 64), (3, 3, 128), (6, 1, 64), (40, 1, 128)])
def test_single_tokens(hq, hkv, dim, page, fp8):
    """One new token per request: lengths of one, of a tile less and more than whole, and split ranges."""
    lens = [1, 2, 31, 32, 33, 127, 128, 129, 255, 257, 1000, 2049, 0, 4111]
    new = [1] * len(lens)
    announce(f"paged attention, single tokens {hq}/{hkv} x {dim}, page {page}, fp8 {fp8}")
    c = make_pages(lens, page, hkv, dim, fp8, seed=dim + page)
    q = make_q(new, hq, dim, 1, packed=False)
    out = run_attention(c, q, lens, new, packed=False)
    check_attention(c, q, out, lens, new, packed=False)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 4, 128, 16), (8, 2, 256, 32), (16, 4, 64, 128), (5, 5, 128, 16),
                                             (6, 1, 256, 64)])
def test_packed_suffixes(hq, hkv, dim, page, gated, fp8):
    """Suffixes of unequal length behind prefixes of unequal length, requests without new tokens or
    without a prefix among them."""
    new = [40, 1, 0, 7, 133, 300, 64]
    cached = [500, 1000, 77, 0, 1, 2500, 64]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"paged attention, packed suffixes {hq}/{hkv} x {dim}, page {page}, gated {gated}, fp8 {fp8}")
    c = make_pages(lens, page, hkv, dim, fp8, seed=dim + page)
    q = make_q(new, hq, dim, 2)
    gate = make_q(new, hq, dim, 3) if gated else None
    out = run_attention(c, q, lens, new, gate=gate)
    check_attention(c, q, out, lens, new, gate=gate)


@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 64), (3, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("new", [[5000], [2900, 33, 700, 1], [1333, 1400, 1500]])
def test_prompts_of_many_row_tiles(new, hq, hkv, dim):
    """Row tiles that fill several rounds of workgroups and are dealt to the XCDs: every one once."""
    announce(f"paged attention, prompts {new}, {hq}/{hkv} x {dim}")
    c = make_pages(new, 64, hkv, dim, False, seed=26)
    q = make_q(new, hq, dim, 27)
    out = run_attention(c, q, new, new)
    check_attention(c, q, out, new, new)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_either_kernel_takes_any_lengths(dim, few):
    """max_seqlen chooses the kernel and bounds nothing: the few-rows kernel on long suffixes, the other
    one on single tokens."""
    new, cached = [200, 1, 30], [700, 900, 0]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"paged attention, few rows kernel {few} x {dim}")
    c = make_pages(lens, 16, 2, dim, False, seed=5)
    q = make_q(new, 8, dim, 4)
    out = run_attention(c, q, lens, new, max_seqlen=1 if few else 231)
    check_attention(c, q, out, lens, new)


@pytest.mark.parametrize("group,hkv", [(1, 2), (5, 2), (7, 1), (13, 1), (31, 1), (33, 1), (127, 1), (129, 1), (1000, 1),
                                       (2048, 1)])
def test_groups_of_every_kind(group, hkv):
    """Query heads per key head that divide no tile: rows change their token inside one, or a token fills many."""
    new, cached = [1, 3, 10], [300, 0, 90]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"paged attention, {group} query heads per key head")
    c = make_pages(lens, 16, hkv, 64, False, seed=16)
    q = make_q(new, group * hkv, 64, 17)
    out = run_attention(c, q, lens, new)
    check_attention(c, q, out, lens, new)


@pytest.mark.parametrize("n", [1, 40])
def test_many_requests(n):
    """More requests than lanes of a wavefront, ragged, the longest last."""
    lens = [n + (i * 37) % 300 for i in range(149)] + [6000]
    new = [n] * 150
    announce(f"paged attention, 150 requests of {n}")
    c = make_pages(lens, 16, 2, 64, False, seed=6)
    q = make_q(new, 8, 64, 5, packed=False)
    out = run_attention(c, q, lens, new, packed=False)
    check_attention(c, q, out, lens, new, packed=False)


@pytest.mark.parametrize("n", [1, 50])
def test_rows_that_see_no_key_are_zeros(n):
    """Requests shorter than their new tokens, of no key, or all of whose keys are on no page."""
    lens = [n - 1, 0, 100, 70]
    announce(f"paged attention, rows without keys, {n} new")
    c = make_pages([120] * 4, 16, 4, 128, False, seed=7)
    c["table"][2] = -1
    c["table"][3, 1] = 1 << 20   # keys 16 .. 31 on no page
    c["table"][3, 4] = -7        # keys 64 .. 79
    q = make_q([n] * 4, 16, 128, 6, packed=False)
    out = run_attention(c, q, lens, [n] * 4, packed=False)
    assert out[1].abs().max() == 0 and out[2].abs().max() == 0 and out[0, :, 0].abs().max() == 0
    check_attention(c, q, out, lens, [n] * 4, packed=False)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 20, 100])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nothing_masked_reaches_a_row(dim, n, fp8):
    """NaN and infinities behind a request's last key, in pages of nobody, and in keys and values of later
    tokens: rows that do not see them are as without them."""
    lens = [n + 75, n + 201]
    announce(f"paged attention, NaN in masked places x {dim}, {n} new, fp8 {fp8}")
    c = make_pages(lens, 16, 2, dim, fp8, seed=8)
    q = make_q([n] * 2, 8, dim, 7, packed=False)
    clean = run_attention(c, q, lens, [n] * 2, packed=False)
    odd = torch.full((dim,), float("nan"), device="cuda")
    if not fp8:
        odd[::3] = float("inf")
        odd[1::3] = -float("inf")
    odd = odd.to(c["k"].dtype)
    for name in ("k", "v"):
        pool = c[name]
        owned = torch.zeros(pool.shape[0], dtype=torch.bool, device="cuda")
        owned[c["table"][c["table"] >= 0].long()] = True
        for p in (~owned).nonzero().flatten().tolist():
            pool[p] = odd
        for r, n_keys in enumerate(lens):
            last = c["table"][r, (n_keys - 1) // 16]
            if n_keys % 16:
                pool[last, :, n_keys % 16:] = odd
            for key in range(n_keys - n // 2, n_keys):  # the later half of the new tokens
                pool[c["table"][r, key // 16], :, key % 16] = odd
    out = run_attention(c, q, lens, [n] * 2, packed=False)
    first = n - n // 2
    assert torch.equal(out[:, :, :first].view(torch.int16), clean[:, :, :first].view(torch.int16))
    assert not torch.isfinite(out[:, :, first:]).any() if n > 1 else True


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [7, 12])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nothing_masked_reaches_a_row_of_middling_requests(dim, n, fp8):
    """The same with 28 and 48 rows of a key head: two tiles of the few-rows kernels."""
    test_nothing_masked_reaches_a_row(dim, n, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,dim", [(16, 4, 128), (8, 2, 256), (16, 4, 64)])
@pytest.mark.parametrize("new", [[8] * 5, [9, 16, 1, 0, 12], [32], [33], [16, 17]])
def test_requests_of_a_few_tokens(new, hq, hkv, dim, fp8):
    """Rows of a key head around every kernel's bounds (32, 64, 128 in all)."""
    announce(f"paged attention, {new} new, {hq}/{hkv} x {dim}, fp8 {fp8}")
    lens = [n + c for n, c in zip(new, [1500, 0, 700, 33, 2100])]
    c = make_pages(lens, 32, hkv, dim, fp8, seed=18)
    q = make_q(new, hq, dim, 19)
    out = run_attention(c, q, lens, new)
    check_attention(c, q, out, lens, new)


def test_a_seen_infinity_reaches_its_feature_alone():
    """An infinite value of a key that a row sees, next to rows that do not see it."""
    announce("paged attention, a seen infinity")
    n, lens = 50, [90]
    c = make_pages(lens, 16, 1, 64, False, seed=9)
    q = make_q([n], 4, 64, 8, packed=False)
    clean = run_attention(c, q, lens, [n], packed=False)
    key = 70  # the token of row 30
    c["v"][c["table"][0, key // 16], 0, key % 16, 5] = float("inf")
    out = run_attention(c, q, lens, [n], packed=False)
    assert (out[0, :, 30:, 5] == float("inf")).all()
    out[0, :, 30:, 5] = clean[0, :, 30:, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("fp8", [False, True])
def test_strided_views(fp8):
    """Heads-inside pages, rows of a wider pool, q and gate as halves of one projection, page tables of a
    wider table, a scale of the caller's."""
    announce(f"paged attention, strided views, fp8 {fp8}")
    lens, new = [300, 45], [33, 45]
    c = make_pages(lens, 32, 4, 128, fp8, seed=10)
    for name in ("k", "v"):
        pool = c[name]
        wide = torch.zeros((pool.shape[0], 32, 4, 160), dtype=pool.dtype, device="cuda")  # [page, row, head, wider]
        view = wide[..., 16:144].permute(0, 2, 1, 3)
        view.copy_(pool)
        c[name] = view
        if fp8:
            ws = torch.zeros((pool.shape[0], 5, 40), dtype=torch.uint8, device="cuda")[:, 1:, 3:35]
            ws.copy_(c[name + "s"])
            c[name + "s"] = ws
    table = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    table[:, 3:3 + c["table"].shape[1]] = c["table"]
    c["table"] = table[:, 3:3 + c["table"].shape[1]]
    qg = make_q(new, 16, 256, 9)
    q, gate = qg[..., :128], qg[..., 128:]
    out = run_attention(c, q, lens, new, gate=gate, scale=0.05)
    check_attention(c, q, out, lens, new, gate=gate, scale=0.05)


@pytest.mark.parametrize("n", [1, 64])
def test_offsets_beyond_32_bits(n):
    """Pages that begin more than 2^32 bytes into their pool."""
    announce(f"paged attention, far pages, {n} new")
    lens, page = [700], 64
    c = make_pages(lens, page, 4, 128, False, seed=11)
    used = c["k"].shape[0]
    far = (2 ** 32 + 2 ** 30) // (4 * page * 128 * 2)
    for name in ("k", "v"):
        pool = torch.empty((far + used, 4, page, 128), dtype=torch.bfloat16, device="cuda")
        pool[far:] = c[name]
        c[name] = pool
    c["table"] = torch.where(c["table"] >= 0, c["table"] + far, c["table"])
    q = make_q([n], 16, 128, 10, packed=False)
    out = run_attention(c, q, lens, [n], packed=False)
    check_attention(c, q, out, lens, [n], packed=False)


def test_rows_behind_the_last_request_stay():
    """A captured step of a fixed size with fewer live tokens: the output's rows behind them are not written."""
    announce("paged attention, rows behind the last request")
    from fastdecisions_amd import _cache_lib, _lib
    from fastdecisions_amd.paged_kv_kernel import check_cache
    import ctypes
    lens, new = [200, 333], [3, 50]
    c = make_pages(lens, 16, 4, 128, False, seed=12)
    q = make_q([80], 16, 128, 11)
    out = torch.full((1, 80, 16, 128), 7.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    cu, lens_t = ints([0, 3, 53]), ints(lens)
    cache = _cache_lib.PagedCache.from_buffer_copy(check_cache(c["k"], c["v"], c["table"], lens_t, None, None, 2))
    lib = _cache_lib.lib()
    size = lib.fd_paged_gqa_workspace_bytes(1, 16, 4, 80, 128, 16, cache.max_pages, 2, 50)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    _cache_lib.check("fd_paged_gqa_fwd", lib.fd_paged_gqa_fwd(
        q.data_ptr(), ctypes.byref(cache), None, out.data_ptr(), _lib.strides4(q), None, _lib.strides4(out), 1, 16, 80,
        128 ** -0.5, cu.data_ptr(), 2, 50, work.data_ptr(), size, _lib.stream_handle(q.device)))
    assert (out[:, :, 53:] == 7.0).all()
    check_attention(c, q, out, lens, new)


@pytest.mark.parametrize("cu", [[0, 90, 40, 80], [5, 5, 70, 500], [-3, 20, 20, 80], [80, 60, 40, 0]])
def test_malformed_offsets_stay_inside(cu):
    """Offset tables that are not ascending or leave the T axis: whatever is computed, every access stays
    inside the tensors (rows are clamped) and a well-formed call afterwards is right."""
    announce(f"paged attention, offsets {cu}")
    lens = [3000, 500, 90]
    c = make_pages(lens, 16, 4, 64, False, seed=13)
    q = make_q([80], 16, 64, 12)
    run_attention(c, q, lens, [80], cu_seqlens=ints(cu), max_seqlen=80)
    new = [30, 30, 20]
    out = run_attention(c, q, lens, new)
    check_attention(c, q, out, lens, new)


@pytest.mark.parametrize("n", [1, 48])
def test_replayed_with_other_lengths(n):
    """A captured call replayed as the requests grow: grids and workspaces come from sizes, not lengths."""
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    announce(f"paged attention, captured, {n} new")
    c = make_pages([5000, 5000], 16, 4, 128, False, seed=14)
    lens = ints([n, n])
    q = make_q([n, n], 16, 128, 13, packed=False)
    call = lambda: paged_gqa_attention(q, c["k"], c["v"], c["table"], lens)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for now in ([n, 70 + n], [4999, 5000], [n, n], [1200, 3100]):
        lens.copy_(ints(now))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        check_attention(c, q, out, now, [n, n], packed=False)


def test_two_streams_at_once():
    """Calls that overlap on two streams, each with its own workspace."""
    announce("paged attention, two streams")
    lens, new = [4000, 2500, 3100], [1, 1, 1]
    cs = [make_pages(lens, 16, 4, 128, fp8, seed=15) for fp8 in (False, True)]
    qs = [make_q(new, 16, 128, 14 + i, packed=False) for i in range(2)]
    want = [run_attention(c, q, lens, new, packed=False) for c, q in zip(cs, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    lens_t = ints(lens)
    torch.cuda.synchronize()
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                c = cs[i]
                got[i].append(paged_gqa_attention(qs[i], c["k"], c["v"], c["table"], lens_t, **scales(c)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


# ---------------------------------------------------------------- writing and reading

def new_rows(new, heads, dim, seed, packed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (1, sum(new), heads, dim) if packed else (len(new), new[0], heads, dim)
    size = torch.exp2(torch.randint(-20, 20, (*shape[:3], 1), generator=gen, device="cuda").float())
    return (torch.randn(shape, generator=gen, device="cuda") * size).to(torch.bfloat16).transpose(1, 2)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,dim,page", [(4, 128, 16), (2, 256, 64), (3, 64, 256), (1, 128, 32)])
@pytest.mark.parametrize("packed", [True, False])
def test_written_rows(packed, heads, dim, page, fp8):
    """New rows where they belong, bit for bit, and nothing else touched; absent pages skipped."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_write
    new = [33, 1, 0, 200, 5] if packed else [17] * 4
    cached = [20, 511, 9, 0, 250][:len(new)]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"paged write {heads} x {dim}, page {page}, packed {packed}, fp8 {fp8}")
    c = make_pages(lens, page, heads, dim, fp8, seed=20)
    lost = len(new) - 2                        # a request one of whose pages is not there
    c["table"][lost, 0] = 1 << 30
    k, v = (new_rows(new, heads, dim, 21 + i, packed) for i in range(2))
    want = {name: c[name].clone() for name in ("k", "v")}
    wants = {name: None if c[name] is None else c[name].clone() for name in ("ks", "vs")}
    at = starts(new)
    for name, x in (("k", k), ("v", v)):
        for r, n in enumerate(new):
            pos = lens[r] - n + torch.arange(n, device="cuda")
            pages = c["table"][r].long()[pos // page]
            keep = (pages >= 0) & (pages < c["k"].shape[0])
            y = (x[0, :, at[r]:at[r + 1]] if packed else x[r]).transpose(0, 1)[keep]
            pages, within = pages[keep], (pos % page)[keep]
            if fp8:
                codes, scale = e4m3(y.double())
                want[name].view(torch.uint8)[pages, :, within] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
                wants[name + "s"][pages, :, within] = scale
            else:
                want[name][pages, :, within] = y
    paged_kv_write(k, v, c["k"], c["v"], c["table"], ints(lens), cu_seqlens=ints(at) if packed else None, **scales(c))
    kind = torch.uint8 if fp8 else torch.int16
    for name in ("k", "v"):
        assert torch.equal(c[name].view(kind), want[name].view(kind)), name
        if fp8:
            assert torch.equal(c[name + "s"], wants[name + "s"]), name


def test_every_row_size_is_quantised_by_the_rule():
    """Rows whose largest value is each bf16 magnitude in turn; zeros, subnormals, infinities, NaN."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_write
    announce("paged write, e4m3 scales of every bf16 magnitude")
    bits = torch.arange(0, 0x7f80, dtype=torch.int32)
    n = bits.numel()
    top = bits.to(torch.int16).view(torch.bfloat16).cuda()
    gen = torch.Generator(device="cuda").manual_seed(22)
    x = (top.float()[:, None] * (torch.rand((n, 64), generator=gen, device="cuda") * 2 - 1)).to(torch.bfloat16)
    x = torch.where(x.abs() > top[:, None], top[:, None], x)
    x[:, 5] = top
    page = 256
    pages = -(-n // page)
    k = torch.zeros((pages, 1, page, 64), dtype=torch.float8_e4m3fn, device="cuda")
    v, ks = torch.zeros_like(k), torch.zeros((pages, 1, page), dtype=torch.uint8, device="cuda")
    vs = torch.zeros_like(ks)
    odd = x.clone()
    odd[:, 9], odd[:, 10], odd[:, 11] = float("inf"), -float("inf"), float("nan")
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    paged_kv_write(x[None, None], odd[None, None], k, v, table, ints([n]), k_scale=ks, v_scale=vs)
    codes, scale = e4m3(x.double())
    assert torch.equal(ks.flatten()[:n], scale)
    assert torch.equal(k.reshape(-1, 64)[:n].double(), codes)
    codes, scale = e4m3(odd.double())
    assert torch.equal(vs.flatten()[:n], scale)
    got = v.reshape(-1, 64)[:n].double()
    assert torch.equal(torch.isnan(got), torch.isnan(odd)) and torch.equal(got.nan_to_num(0), codes.nan_to_num(0))
    # half a step of the code: 2^-4 of the value, or half of the smallest step 2^-9 of the scale
    back = k.reshape(-1, 64)[:n].double() * pow2(ks.flatten()[:n])[:, None]
    assert ((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, pow2(ks.flatten()[:n])[:, None] * 2.0 ** -10)).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,dim,page", [(4, 128, 16), (2, 256, 64), (3, 64, 256)])
def test_read_back(heads, dim, page, fp8):
    """The first rows of every request as bf16; zeros on absent pages and past the table; rows behind the
    last request stay."""
    from fastdecisions_amd import _cache_lib, _lib
    from fastdecisions_amd.paged_kv_kernel import check_cache, paged_kv_read
    import ctypes
    announce(f"paged read {heads} x {dim}, page {page}, fp8 {fp8}")
    lens = [1, 700, 0, 33, 300]
    c = make_pages(lens, page, heads, dim, fp8, seed=23, spare_entries=0)
    c["table"][4, 0] = -1
    ask = [1, 650, 0, 33, c["table"].shape[1] * page + 9]   # the last one: beyond its table
    at, total = starts(ask), sum(ask)
    k, v = paged_kv_read(c["k"], c["v"], c["table"], ints(at), total, **scales(c))
    assert k.shape == v.shape == (1, heads, total, dim) and k.dtype == torch.bfloat16
    for name, got in (("k", k), ("v", v)):
        for r, n in enumerate(ask):
            m = min(n, c["table"].shape[1] * page)
            x, there = rows(c, name, r, m)
            want = torch.where(there[None, :, None], x, 0.0).to(torch.bfloat16)
            assert torch.equal(got[0, :, at[r]:at[r] + m], want), (name, r)
            assert (got[0, :, at[r] + m:at[r + 1]] == 0).all()
    out = torch.full((total + 5, heads, dim), 3.0, dtype=torch.bfloat16, device="cuda")
    cache = _cache_lib.PagedCache.from_buffer_copy(check_cache(c["k"], c["v"], c["table"], None, c["ks"], c["vs"], len(ask)))
    s2 = (ctypes.c_int64 * 2)(dim, heads * dim)
    cu = ints(at)
    _cache_lib.check("fd_paged_kv_read", _cache_lib.lib().fd_paged_kv_read(
        ctypes.byref(cache), out.data_ptr(), out.data_ptr(), s2, s2, total + 5, cu.data_ptr(), len(ask),
        _lib.stream_handle(out.device)))
    assert (out[total:] == 3.0).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_calls(dim, fp8):
    """Calls in which a thread writes and reads several rows: bits as of the short calls' one, packed requests of
    every length, a request without tokens among them, a last workgroup that is not full."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    heads, page = 1024 // dim, 32
    new = [7000, 1, 0, 33, 6001, 4200]
    cached = [20, 511, 9, 0, 250, 1]
    lens = [a + b for a, b in zip(cached, new)]
    announce(f"paged write and read, long calls {heads} x {dim}, fp8 {fp8}")
    c = make_pages(lens, page, heads, dim, fp8, seed=24)
    k, v = (new_rows(new, heads, dim, 25 + i, True) for i in range(2))
    at = starts(new)
    paged_kv_write(k, v, c["k"], c["v"], c["table"], ints(lens), cu_seqlens=ints(at), **scales(c))
    all_at = starts(lens)
    got = paged_kv_read(c["k"], c["v"], c["table"], ints(all_at), all_at[-1], **scales(c))
    for name, x, out in zip(("k", "v"), (k, v), got):
        for r, n in enumerate(new):
            want, there = rows(c, name, r, lens[r])
            assert there.all() and torch.equal(out[0, :, all_at[r]:all_at[r + 1]], want.to(torch.bfloat16)), (name, r)
            mine = x[0, :, at[r]:at[r + 1]]
            if fp8:
                codes, scale = e4m3(mine.double())
                mine = (codes * pow2(scale)[..., None]).to(torch.bfloat16)
            assert torch.equal(out[0, :, all_at[r] + cached[r]:all_at[r + 1]], mine), (name, r)


def test_written_then_attended_then_read():
    """A run as a program makes it: a prompt in pieces and then tokens one by one, quantised, equal to
    attention over everything at once."""
    from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    announce("paged write, attention and read together")
    total, heads, dim, page = 700, 4, 128, 16
    c = make_pages([total], page, heads, dim, True, seed=24)
    k, v = (new_rows([total], heads, dim, 25 + i, True).clamp(-3, 3) for i in range(2))
    q = make_q([total], 16, dim, 27)
    outs, done = [], 0
    for n in (300, 1, 1, 257, 64, 1, 76):
        done += n
        part = slice(done - n, done)
        lens = ints([done])
        paged_kv_write(k[:, :, part], v[:, :, part], c["k"], c["v"], c["table"], lens, **scales(c))
        outs.append(paged_gqa_attention(q[:, :, part], c["k"], c["v"], c["table"], lens, **scales(c)))
    assert done == total
    check_attention(c, q, torch.cat(outs, dim=2), [total], [total])
    dk, dv = paged_kv_read(c["k"], c["v"], c["table"], ints([0, total]), total, **scales(c))
    for got, x in ((dk, k), (dv, v)):
        codes, scale = e4m3(x[0].double())
        assert torch.equal(got[0].double(), codes * pow2(scale)[..., None])


@pytest.mark.parametrize("fp8", [False, True])
def test_a_run_on_another_stream(fp8):
    """Write, attend and read on a stream of the caller's, with work of the default stream going on: the bits of
    the same run on the default stream."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
    announce(f"paged cache, a run on another stream, fp8 {fp8}")
    new, lens = [70, 1, 300], [900, 2000, 300]

    def run():
        c = make_pages(lens, 32, 4, 128, fp8, seed=28)
        k, v = (new_rows(new, 4, 128, 29 + i, True) for i in range(2))
        q = make_q(new, 16, 128, 31)
        paged_kv_write(k, v, c["k"], c["v"], c["table"], ints(lens), cu_seqlens=ints(starts(new)), **scales(c))
        out = run_attention(c, q, lens, new)
        return [out, *paged_kv_read(c["k"], c["v"], c["table"], ints(starts(lens)), sum(lens), **scales(c))]
    want = run()
    side, busy = torch.cuda.Stream(), torch.zeros(1 << 26, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        busy.add_(1.0)
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_reading_nothing():
    """A request without keys: empty tensors, the pool untouched."""
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read
    announce("paged read, no rows")
    c = make_pages([40], 16, 2, 64, False, seed=32)
    k, v = paged_kv_read(c["k"], c["v"], c["table"], ints([0, 0]), 0)
    assert k.shape == v.shape == (1, 2, 0, 64) and k.dtype == torch.bfloat16
