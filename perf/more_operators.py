"""Operators that let a decider's cache hold more, as calls that are timed.

A decision service is bounded by what its paged caches hold: prefixes of thousands
of tokens, forked per question.  Keys and values in 4 bits (e2m1 codes, two a byte,
with a power-of-two scale per 32 features: 4.25 bits a value) take about half the
room and the bytes of 8-bit ones, and of a long prefix most keys draw next to no
attention, so that a request can go on with the keys that did.

    store    keys and values of new tokens into 4-bit pages, and what attention then reads of them
    read     4-bit pages back as dense keys and values
    attn     attention of the new tokens of every request over their 4-bit pages
    weights  the attention weight that every cached key draws from the new tokens, added to its sum
             (bf16, e4m3 or 4-bit pages)
    evict    the keys of largest weight and the most recent ones, per key head, moved to pages of their own

    own                   False: plain torch in 32 bits; True: this package's entry points
    listed(), draw(rng)   the cases
    prepare(case, seed)   what a program holds before the call
    run(state)            one pass; returns its outputs
    work(case)            bytes and flops the pass cannot do without
    exact(case, seed)     the outputs in 64 bits
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 32       # features that share a scale of the 4-bit cache
E4M3_MAX = 448.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # values of the codes; bit 3 is the sign
E2M1_TIES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def listed():
    return [
        # one token of one short request: the smallest call of the attention, latency only
        {"name": "attn_token_short", "kind": "attn", "requests": 1, "cached": "189,189", "new": "1,1", "lens_seed": 1,
         "hq": 16, "hkv": 4, "d": 128, "page": 16, "gated": False},
        # a decoding step of 64 requests of a few hundred to 8192 cached tokens, output gate
        {"name": "attn_tokens_64", "kind": "attn", "requests": 64, "cached": "256,8192", "new": "1,1", "lens_seed": 2,
         "hq": 16, "hkv": 4, "d": 128, "page": 64, "gated": True},
        # suffixes (one question each) packed behind long cached prefixes, output gate
        {"name": "attn_suffixes", "kind": "attn", "requests": 6, "cached": "2048,8192", "new": "30,400", "lens_seed": 3,
         "hq": 16, "hkv": 4, "d": 128, "page": 16, "gated": True},
        # the last piece of a long prompt fed in pieces, 8/2 heads of 256
        {"name": "attn_piece_d256", "kind": "attn", "requests": 1, "cached": "6144,6144", "new": "2048,2048",
         "lens_seed": 4, "hq": 8, "hkv": 2, "d": 256, "page": 128, "gated": False},
        # one token each of 64 short requests
        {"name": "store_tokens_64", "kind": "store", "requests": 64, "cached": "16,256", "new": "1,1", "lens_seed": 5,
         "hkv": 4, "d": 128, "page": 16},
        # whole prompts packed into one row
        {"name": "store_prompts", "kind": "store", "requests": 4, "cached": "0,0", "new": "256,8192", "lens_seed": 6,
         "hkv": 4, "d": 128, "page": 64},
        # a short prefix read back
        {"name": "read_short", "kind": "read", "requests": 1, "cached": "611,611", "new": "0,0", "lens_seed": 7,
         "hkv": 2, "d": 256, "page": 16},
        # long prefixes read back
        {"name": "read_prompts", "kind": "read", "requests": 6, "cached": "256,8192", "new": "0,0", "lens_seed": 8,
         "hkv": 4, "d": 128, "page": 64},
        # weights gathered while 64 requests decode, 4-bit cache
        {"name": "weights_tokens_64", "kind": "weights", "requests": 64, "cached": "256,8192", "new": "1,1",
         "lens_seed": 9, "hq": 16, "hkv": 4, "d": 128, "page": 64, "held": "e2m1", "last": 0},
        # weights gathered over the last piece of a long prompt, bf16 cache
        {"name": "weights_piece", "kind": "weights", "requests": 1, "cached": "2048,2048", "new": "2900,2900",
         "lens_seed": 10, "hq": 16, "hkv": 4, "d": 128, "page": 64, "held": "bf16", "last": 0},
        # one prefix of a few hundred tokens cut to 256 keys, bf16 cache: latency only
        {"name": "evict_short", "kind": "evict", "requests": 1, "cached": "700,700", "new": "0,0", "lens_seed": 11,
         "hkv": 4, "d": 128, "page": 16, "held": "bf16", "keep": 256, "recent": 32},
        # long prefixes of several requests cut to 2048 keys each, 8-bit cache
        {"name": "evict_prompts", "kind": "evict", "requests": 12, "cached": "1500,16384", "new": "0,0", "lens_seed": 12,
         "hkv": 4, "d": 128, "page": 64, "held": "e4m3", "keep": 2048, "recent": 128},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "store", "read", "weights", "weights", "evict"])
    hq, hkv, d = rng.choice([(16, 4, 128), (16, 4, 128), (8, 2, 256), (16, 4, 64), (8, 8, 128), (6, 1, 128)])
    case = {"kind": kind, "lens_seed": rng.randint(1, 1 << 30), "hkv": hkv, "d": d, "page": rng.choice([16, 16, 32, 64, 128, 256])}
    if kind in ("store", "read"):
        top = _log_int(rng, 2, 8192)
        case["requests"] = _log_int(rng, 1, max(1, min(64, 16000 // top)))
        if kind == "read":
            return {**case, "cached": f"1,{top}", "new": "0,0"}
        return {**case, "cached": f"1,{_log_int(rng, 2, 256)}", "new": f"1,{top}"}
    if kind != "attn":
        case["held"] = rng.choice(["bf16", "e4m3", "e2m1"])
    if kind == "evict":
        top = _log_int(rng, 64, 16384)
        keep = _log_int(rng, 16, min(top, 2048))
        return {**case, "requests": _log_int(rng, 1, max(1, min(64, 64000 // top))), "cached": f"{max(1, top // 16)},{top}",
                "new": "0,0", "keep": keep, "recent": rng.choice([0, rng.randint(0, keep)])}
    case["hq"] = hq
    if kind == "attn":
        case["gated"] = rng.random() < 0.5
    top = _log_int(rng, 16, 8192)
    if rng.random() < 0.4:  # single tokens
        return {**case, "requests": _log_int(rng, 1, 64), "cached": f"1,{top}", "new": "1,1",
                **({"last": 0} if kind == "weights" else {})}
    new = _log_int(rng, 2, 1200)
    case |= {"requests": rng.randint(1, 8 if new <= 100 else 4 if new <= 300 else 1), "cached": f"1,{top}", "new": f"1,{new}"}
    if kind == "weights":
        case["last"] = rng.choice([0, 0, _log_int(rng, 1, 64)])
    return case


# ---------------------------------------------------------------- sizes

def _lens(case):
    """(cached tokens, new tokens) of every request: log-uniform between the case's bounds."""
    rng = random.Random(case["lens_seed"])

    def some(bounds):
        lo, hi = (int(b) for b in bounds.split(","))
        return [lo if lo == hi else _log_int(rng, lo, hi) for _ in range(case["requests"])]
    return some(case["cached"]), some(case["new"])


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _row_bytes(case):
    """Bytes of one cached row of K or V."""
    d, held = case["d"], case.get("held", "e2m1")
    return 2 * d if held == "bf16" else d + 1 if held == "e4m3" else d // 2 + d // BLOCK


def work(case):
    cached, new = _lens(case)
    hkv, d, total = case["hkv"], case["d"], sum(new)
    held = hkv * _row_bytes(case)
    keys = sum(cached) + total
    if case["kind"] == "store":  # rows in and pages out, then pages in and rows out
        return {"bytes": 2 * total * (hkv * d * 2 + held) + 2 * keys * (hkv * d * 2 + held), "flops": 4 * total * hkv * d}
    if case["kind"] == "read":
        return {"bytes": 2 * keys * (hkv * d * 2 + held), "flops": 2 * keys * hkv * d}
    if case["kind"] == "evict":
        left = sum(min(n, case["keep"]) for n in cached)
        return {"bytes": 4 * hkv * (keys + left) + 4 * left * held + 4 * hkv * left, "flops": keys * hkv}
    last = case.get("last") or max(new)
    seen = [min(m, last) for m in new]   # tokens whose rows count
    pairs = sum(m * (c + n) - m * (m - 1) // 2 for c, n, m in zip(cached, new, seen))
    if case["kind"] == "weights":
        return {"bytes": keys * held + sum(seen) * case["hq"] * d * 2 + 8 * hkv * keys, "flops": 2 * case["hq"] * d * pairs}
    return {"bytes": 2 * keys * held + total * case["hq"] * d * 2 * (3 if case["gated"] else 2),
            "flops": 4 * case["hq"] * d * pairs}


# ---------------------------------------------------------------- inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _pages(case, held, gen, more=0):
    """A pool a quarter larger than the requests need, its pages dealt to them in random order:
    (page table [requests, most pages + 1] with -1 where a request has no page, `more` pages of
    nobody's for each request, pool size)."""
    need = [-(-t // case["page"]) for t in held]
    pool = sum(need) + more * len(need) + sum(need) // 4 + 1
    order = torch.randperm(pool, generator=gen, device=DEV).tolist()
    at = _starts(need)
    table = [order[a:b] + [-1] * (max(need) + 1 - (b - a)) for a, b in zip(at, at[1:])]
    spare = [order[at[-1] + more * r:at[-1] + more * (r + 1)] for r in range(len(need))]
    return _ints(table), spare, pool


def _pool(case, gen, shape, held):
    """Keys or values as the quantiser leaves them: (pool, scales or None)."""
    *lead, d = shape
    if held == "bf16":
        return _normal(gen, *shape), None
    if held == "e4m3":  # the largest code of each row lies between half the range and its end
        codes = _normal(gen, *shape, std=100.0, dtype=torch.float32).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return codes, torch.randint(118, 122, lead, generator=gen, device=DEV, dtype=torch.uint8)
    x = torch.randn(shape, generator=gen, device=DEV) * 2.0
    scale = torch.randint(125, 128, (*lead, d // BLOCK), generator=gen, device=DEV, dtype=torch.uint8)
    return _pack(_codes(x)), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    cached, new = _lens(case)
    n, total = len(new), sum(new)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    held = [a + b for a, b in zip(cached, new)]
    packed = max(new) != min(new) or kind == "read"
    s = {"case": case, "new": new, "held": held, "max_new": max(new), "max_held": max(held), "total": sum(held),
         "cu": _ints(_starts(new)) if packed else None, "lens": _ints(held)}
    s["table"], spare, pool = _pages(case, held, gen, -(-case["keep"] // page) if kind == "evict" else 0)
    shape = (pool, hkv, page, d)
    if kind == "store":
        s["kc"], s["vc"] = (torch.zeros((*shape[:3], d // 2), dtype=torch.uint8, device=DEV).view(torch.float4_e2m1fn_x2)
                            for _ in range(2))
        s["ks"], s["vs"] = (torch.full((*shape[:3], d // BLOCK), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
        s["all"] = _ints(_starts(held))
        rows = (1, total) if packed else (n, new[0])
        # projections as the layer makes them: [B, T, H, D], read as [B, H, T, D]; features of unequal size
        s["k"], s["v"] = ((_normal(gen, *rows, hkv, d) * torch.exp2(torch.randint(-3, 3, (*rows, hkv, d // 16), generator=gen,
                                                                                  device=DEV)).to(torch.bfloat16)
                           .repeat_interleave(16, dim=-1)).transpose(1, 2) for _ in range(2))
        return s
    s["kc"], s["ks"] = _pool(case, gen, shape, case.get("held", "e2m1"))
    if kind != "weights":
        s["vc"], s["vs"] = _pool(case, gen, shape, case.get("held", "e2m1"))
    if kind == "read":
        s["cu"] = _ints(_starts(held))
        return s
    if kind in ("weights", "evict"):  # rows of a larger pool, as a cache's slots
        width = s["table"].shape[1] * page
        s["rows"] = torch.randperm(n + 3, generator=gen, device=DEV)[:n].to(torch.int32)
        s["weights"] = torch.zeros((n + 3, hkv, width), device=DEV)
    if kind == "evict":  # most keys have drawn little, some a lot, some nothing
        s["weights"].copy_(torch.exp(torch.randn(s["weights"].shape, generator=gen, device=DEV) * 2.0 - 2.0))
        s["weights"] *= torch.rand(s["weights"].shape, generator=gen, device=DEV) > 0.1
        s["new_table"], s["weights_out"] = _ints(spare), torch.zeros_like(s["weights"])
        s["left"] = [min(m, case["keep"]) for m in held]
        s["cu_left"] = _ints(_starts(s["left"]))
        return s
    hq = case["hq"]
    rows = (1, total) if packed else (n, new[0])
    s["q"] = _normal(gen, *rows, hq, d, std=1.5).transpose(1, 2)
    s["gate"] = _normal(gen, *rows, hq, d).transpose(1, 2) if case.get("gated") else None
    return s


# ---------------------------------------------------------------- this package's entry points

def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    packed = {} if s["cu"] is None else {"cu_seqlens": s["cu"], "max_seqlen": s["max_new"]}
    if kind == "attn":
        from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
        return paged_gqa_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], k_scale=s["ks"], v_scale=s["vs"],
                                   gate=s["gate"], **packed)
    if kind == "store":
        from fastdecisions_amd.paged_kv_kernel import paged_kv_read, paged_kv_write
        paged_kv_write(s["k"], s["v"], s["kc"], s["vc"], s["table"], s["lens"], k_scale=s["ks"], v_scale=s["vs"],
                       cu_seqlens=s["cu"])
        return [*paged_kv_read(s["kc"], s["vc"], s["table"], s["all"], s["total"], k_scale=s["ks"], v_scale=s["vs"]),
                s["ks"], s["vs"]]
    if kind == "read":
        from fastdecisions_amd.paged_kv_kernel import paged_kv_read
        return list(paged_kv_read(s["kc"], s["vc"], s["table"], s["cu"], s["total"], k_scale=s["ks"], v_scale=s["vs"]))
    if kind == "weights":
        from fastdecisions_amd.paged_evict_kernel import paged_key_weights
        paged_key_weights(s["q"], s["kc"], s["table"], s["lens"], s["weights"], k_scale=s["ks"], row_indices=s["rows"],
                          last=case["last"] or None, **packed)
        return s["weights"]
    from fastdecisions_amd.paged_evict_kernel import paged_kv_evict
    kept, left = paged_kv_evict(s["kc"], s["vc"], s["table"], s["lens"], s["weights"], s["new_table"], case["keep"],
                                recent=case["recent"], k_scale=s["ks"], v_scale=s["vs"], weights_out=s["weights_out"],
                                row_indices=s["rows"])
    if case["held"] != "e2m1":
        return [kept, left, s["weights_out"], s["kc"], s["vc"], s["ks"], s["vs"]]
    from fastdecisions_amd.paged_kv_kernel import paged_kv_read  # 4-bit rows as the values they stand for
    return [kept, left, s["weights_out"], *paged_kv_read(s["kc"], s["vc"], s["new_table"], s["cu_left"], sum(s["left"]),
                                                         k_scale=s["ks"], v_scale=s["vs"])]


# ---------------------------------------------------------------- plain forms

def _pow2(byte):
    """2^(byte - 127) in 32 bits, exactly."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _codes(x):
    """Nearest e2m1 code of each value in [-6, 6], ties to the even code, sign in bit 3."""
    a = x.abs()
    ties = torch.tensor(E2M1_TIES, device=DEV)
    low, high = torch.bucketize(a, ties), torch.bucketize(a, ties, right=True)  # they differ on a tie alone
    code = torch.where((low & 1) == 0, low, high).to(torch.uint8)
    return code | (torch.signbit(x).to(torch.uint8) << 3)


def _pack(code):
    return (code[..., ::2] | (code[..., 1::2] << 4)).view(torch.float4_e2m1fn_x2)


def _unpack(pool):
    byte = pool.view(torch.uint8)
    code = torch.stack([byte & 15, byte >> 4], dim=-1).flatten(-2)
    value = torch.tensor(E2M1, device=DEV)
    return torch.cat([value, -value])[code.long()]


def _values(pool, scale):
    """Rows as the numbers they stand for, in 32 bits."""
    if scale is None:
        return pool.float()
    if pool.dtype == torch.float8_e4m3fn:
        return pool.float() * _pow2(scale)[..., None]
    return _unpack(pool) * _pow2(scale).repeat_interleave(BLOCK, dim=-1)


def _take(pool, index):
    """pool[index] of any element type."""
    small = pool.dtype in (torch.float8_e4m3fn, torch.float4_e2m1fn_x2)
    return pool.view(torch.uint8)[index].view(pool.dtype) if small else pool[index]


def _dense(s, pool, scale, length, table=None):
    """The first `length` keys of every request [requests, heads, length, d] in 32 bits."""
    page = s["case"]["page"]
    table = (s["table"] if table is None else table)[:, :-(-length // page)].long().clamp(min=0)
    x = _values(_take(pool, table), None if scale is None else scale[table])
    n, p, h, _, d = x.shape
    return x.transpose(1, 2).reshape(n, h, p * page, d)[:, :, :length]


def _of(lens):
    """(request, index within it) of every token in packed order."""
    lens = torch.tensor(lens, device=DEV)
    req = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), lens)
    return req, torch.arange(req.numel(), device=DEV) - (torch.cumsum(lens, 0) - lens)[req]


def _probabilities(s, k):
    """exp(score - row maximum) [requests, hq, new, length], where a token sees a key, and their sums."""
    q, lens = s["q"], s["lens"].long()
    n, new, length = lens.numel(), s["max_new"], s["max_held"]
    hq, d = q.shape[1], q.shape[3]
    if s["cu"] is None:
        qd = q.float()
    else:
        req, at = _of(s["new"])
        qd = torch.zeros((n, hq, new, d), device=DEV)
        qd[req, :, at] = q[0].transpose(0, 1).float()
    count = torch.tensor(s["new"], device=DEV)
    last = (lens - count)[:, None] + torch.arange(new, device=DEV)      # position of each new token
    keys = torch.arange(length, device=DEV)
    seen = keys <= torch.minimum(last, lens[:, None] - 1)[..., None]    # [requests, new, length]
    p = qd.reshape(n, k.shape[1], -1, d) @ k.transpose(2, 3)
    p = (p * d ** -0.5).reshape(n, hq, new, length).masked_fill_(~seen[:, None], float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    return p, p.sum(-1, keepdim=True)


def _plain_attn(s):
    n, new, length = s["lens"].numel(), s["max_new"], s["max_held"]
    hq, d = s["q"].shape[1], s["q"].shape[3]
    k, v = _dense(s, s["kc"], s["ks"], length), _dense(s, s["vc"], s["vs"], length)
    v = torch.where((torch.arange(length, device=DEV) < s["lens"][:, None])[:, None, :, None], v, 0.0)
    p, total = _probabilities(s, k)
    o = (p.reshape(n, k.shape[1], -1, length) @ v).reshape(n, hq, new, d) / total
    if s["cu"] is not None:
        req, at = _of(s["new"])
        o = o[req, :, at].transpose(0, 1)[None]
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(torch.bfloat16)


def _read_back(s, table, lens):
    req, at = _of(lens)
    return [_dense(s, pool, scale, max(lens), table)[req, :, at].to(torch.bfloat16).transpose(0, 1)[None]
            for pool, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]


def _plain_store(s):
    page = s["case"]["page"]
    req, at = _of(s["new"])
    count = torch.tensor(s["new"], device=DEV)
    pos = (s["lens"].long() - count)[req] + at
    slot = s["table"].long()[req, pos // page]
    for x, pool, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3]).float()  # [tokens, heads, d]
        x = x.unflatten(-1, (-1, BLOCK))
        top = x.abs().amax(-1)
        m, e = torch.frexp(top)                                            # top = m 2^e, m in [0.5, 1); 6 = 0.75 2^3
        e = torch.where(top > 0, torch.where(m > 0.75, e - 2, e - 3), 0).clamp(min=-126).to(torch.int32)
        code = _codes((x * _pow2(127 - e)[..., None]).flatten(-2))
        pool.view(torch.uint8)[slot, :, pos % page] = _pack(code).view(torch.uint8)
        scale[slot, :, pos % page] = (e + 127).to(torch.uint8)
    return [*_read_back(s, s["table"], s["held"]), s["ks"], s["vs"]]


def _plain_read(s):
    return _read_back(s, s["table"], s["held"])


def _plain_weights(s):
    case = s["case"]
    n, length = s["lens"].numel(), s["max_held"]
    p, total = _probabilities(s, _dense(s, s["kc"], s["ks"], length))
    count = torch.tensor(s["new"], device=DEV)[:, None]
    at = torch.arange(s["max_new"], device=DEV)
    counts = (at < count) & (at >= count - (case["last"] or s["max_new"]))  # [requests, new]
    p = p.div_(total).masked_fill_(~counts[:, None, :, None], 0.0)
    s["weights"][s["rows"].long(), :, :length] += p.reshape(n, case["hkv"], -1, length).sum(2)
    return s["weights"]


def _plain_evict(s):
    case, page, lens = s["case"], s["case"]["page"], s["lens"].long()
    n, hkv, keep, length = lens.numel(), case["hkv"], case["keep"], s["max_held"]
    w = s["weights"][s["rows"].long(), :, :length]
    pos = torch.arange(length, device=DEV)
    here = (pos < lens[:, None])[:, None].expand(-1, hkv, -1)
    left = lens.clamp(max=keep)
    order = w.masked_fill((pos >= (lens - case["recent"])[:, None])[:, None], float("inf")).masked_fill(~here, -1.0)
    order = torch.sort(order, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(length, device=DEV).expand_as(order)
    chosen = torch.zeros_like(order, dtype=torch.bool).scatter_(2, order, rank < left[:, None, None])
    place = torch.where(chosen, torch.cumsum(chosen, -1) - 1, keep)        # where a kept key goes
    kept = torch.full((n, hkv, keep + 1), -1, dtype=torch.int64, device=DEV)
    kept = kept.scatter_(2, place, pos.expand_as(place))[..., :keep]
    live = kept >= 0
    old = kept.clamp(min=0)
    s["weights_out"][s["rows"].long(), :, :length] = torch.where(here, 0.0, s["weights_out"][s["rows"].long(), :, :length])
    top = min(keep, length)
    s["weights_out"][s["rows"].long(), :, :top] = torch.where(live[..., :top], w.gather(2, old[..., :top]),
                                                              s["weights_out"][s["rows"].long(), :, :top])
    r, h, i = live.nonzero(as_tuple=True)
    j = kept[r, h, i]
    src, dst = s["table"].long()[r, j // page], s["new_table"].long()[r, i // page]
    for pool in (s["kc"], s["vc"], s["ks"], s["vs"]):
        if pool is not None:
            raw = pool if pool.dtype == torch.bfloat16 else pool.view(torch.uint8)
            raw[dst, h, i % page] = raw[src, h, j % page]
    kept, left = kept.to(torch.int32), left.to(torch.int32)
    if case["held"] != "e2m1":
        return [kept, left, s["weights_out"], s["kc"], s["vc"], s["ks"], s["vs"]]
    return [kept, left, s["weights_out"], *_read_back(s, s["new_table"], s["left"])]


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "store": _plain_store, "read": _plain_read, "weights": _plain_weights,
            "evict": _plain_evict}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- in 64 bits

def _two64(e):
    """2^e in 64 bits, exactly (a library's pow need not be)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rows64(s, table, r, pool, scale, length):
    """Keys 0 .. length - 1 of request r, [heads, length, d]."""
    at = torch.arange(length, device=DEV)
    pages, within = table[r].long()[at // s["case"]["page"]], at % s["case"]["page"]
    if pool.dtype == torch.bfloat16:
        return pool[pages, :, within].double().permute(1, 0, 2)
    if pool.dtype == torch.float8_e4m3fn:
        return (pool.double()[pages, :, within] * _two64(scale[pages, :, within].long() - 127)[..., None]).permute(1, 0, 2)
    byte = pool.view(torch.uint8)[pages, :, within].long()
    x = torch.empty((*byte.shape[:2], 2 * byte.shape[2]), dtype=torch.float64, device=DEV)
    for half in range(2):  # sign, two bits of exponent, one of mantissa
        code = (byte >> (4 * half)) & 15
        m, e = code & 1, (code >> 1) & 3
        value = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * _two64(e - 1))
        x[..., half::2] = torch.where(code >= 8, -value, value)
    s64 = _two64(scale[pages, :, within].long() - 127)
    return (x.unflatten(-1, (-1, BLOCK)) * s64[..., None]).flatten(-2).permute(1, 0, 2)


def _exact_e2m1(x):
    """(values held, scale bytes) of rows x [.., d]."""
    x = x.unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp(min=1e-300) / torch.full_like(top, 6.0))), 0.0).clamp(min=-126)
    y = x / _two64(e)[..., None]
    step = _two64(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return (torch.round(y / step) * step * _two64(e)[..., None]).flatten(-2), (e + 127).to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    kind, page, starts = case["kind"], case["page"], _starts(s["new"])
    hkv, d = case["hkv"], case["d"]
    pools = (("kc", "ks"), ("vc", "vs"))
    if kind == "read":
        return [torch.cat([_rows64(s, s["table"], r, s[c], s[e], m) for r, m in enumerate(s["held"])], dim=1)[None]
                for c, e in pools]
    if kind == "store":
        res, scales = [], []
        for x, (c, e) in zip((s["k"], s["v"]), pools):
            scale, rows = s[e].clone(), []
            for r, m in enumerate(s["new"]):
                row, a = (r, 0) if s["cu"] is None else (0, starts[r])
                old = s["held"][r] - m
                pos = old + torch.arange(m, device=DEV)
                y, b = _exact_e2m1(x[row, :, a:a + m].double())
                scale[s["table"][r].long()[pos // page], :, pos % page] = b.transpose(0, 1)
                rows.append(torch.cat([_rows64(s, s["table"], r, s[c], s[e], old), y], dim=1))
            res.append(torch.cat(rows, dim=1)[None])
            scales.append(scale)
        return [*res, *scales]
    if kind == "evict":
        kept = torch.full((len(s["held"]), hkv, case["keep"]), -1, dtype=torch.int32, device=DEV)
        out, rows = s["weights_out"].double(), {"kc": [], "vc": []}
        new = {name: None if s[name] is None else (s[name].double() if name in ("kc", "vc") and case["held"] != "e2m1" else s[name].clone())
               for pair in pools for name in pair}
        for r, m in enumerate(s["held"]):
            at, left = int(s["rows"][r]), s["left"][r]
            out[at, :, :m] = 0.0
            to = torch.arange(left, device=DEV)
            for c, e in pools:
                if case["held"] == "e2m1":
                    rows[c].append(_rows64(s, s["table"], r, s[c], s[e], m))
            for h in range(hkv):
                w = s["weights"][at, h, :m].double().tolist()
                fixed = max(0, m - case["recent"])
                best = sorted(range(fixed), key=lambda j: (-w[j], j))[:max(0, left - (m - fixed))]
                mine = torch.tensor(sorted(best + list(range(fixed, m)))[-left:], device=DEV)
                kept[r, h, :left] = mine.to(torch.int32)
                out[at, h, :left] = s["weights"][at, h, mine].double()
                src, dst = s["table"][r].long()[mine // page], s["new_table"][r].long()[to // page]
                for c, e in pools:
                    if case["held"] == "e2m1":
                        rows[c][-1][h, :left] = rows[c][-1][h, mine]
                        continue
                    new[c][dst, h, to % page] = s[c].double()[src, h, mine % page]
                    if s[e] is not None:
                        new[e][dst, h, to % page] = s[e][src, h, mine % page]
            for c, e in pools:
                if case["held"] == "e2m1":
                    rows[c][-1] = rows[c][-1][:, :left]
        left = _ints(s["left"])
        if case["held"] == "e2m1":
            return [kept, left, out, *(torch.cat(rows[c], dim=1)[None] for c in ("kc", "vc"))]
        return [kept, left, out, new["kc"], new["vc"], new["ks"], new["vs"]]
    hq = case["hq"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV) if kind == "attn" else s["weights"].double()
    for r, m in enumerate(s["new"]):
        row, a = (r, 0) if s["cu"] is None else (0, starts[r])
        length = s["held"][r]
        k = _rows64(s, s["table"], r, s["kc"], s["ks"], length)
        v = _rows64(s, s["table"], r, s["vc"], s["vs"], length) if kind == "attn" else None
        for h in range(hq):
            z = s["q"][row, h, a:a + m].double() @ k[h * hkv // hq].T / math.sqrt(d)
            z += torch.full_like(z, -math.inf).triu(length - m + 1)
            p = torch.softmax(z, dim=-1)
            if kind == "weights":
                first = m - case["last"] if 0 < case["last"] < m else 0
                out[int(s["rows"][r]), h * hkv // hq, :length] += p[first:].sum(0)
                continue
            o = p @ v[h * hkv // hq]
            if s["gate"] is not None:
                o *= torch.sigmoid(s["gate"][row, h, a:a + m].double())
            out[row, h, a:a + m] = o
    return out
