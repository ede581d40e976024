"""Operators that continue a decider request from its caches, as calls that are timed.

A decision service scores many questions over one prefix, feeds long prompts in
pieces and extends requests by a token or a few.  What it keeps between calls is
a paged key/value cache per attention layer (bf16, or e4m3 codes with one
power-of-two scale per token and head) and, per linear-attention layer, the last
rows of the causal conv and the fp32 state of the delta rule.  Five operators
work on them:

    attn    attention of the new tokens of every request over their paged cache
    write   keys and values of new tokens into the pages
    read    the pages back as dense keys and values
    delta   the gated delta rule token by token, from and into its state
    conv    the causal conv + SiLU continued from its state

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
HEAD = 128       # head dim of the linear-attention layers
WIDTH = 4        # taps of the causal conv
E4M3_MAX = 448.0


def listed():
    return [
        # one token of one short request: the smallest call of the attention, latency only
        {"name": "attn_token_short", "kind": "attn", "requests": 1, "cached": "189,189", "new": "1,1", "lens_seed": 1,
         "hq": 16, "hkv": 4, "d": 128, "page": 16, "fp8": False, "gated": False},
        # a decoding step of 64 requests of a few hundred to 8192 cached tokens, 8-bit cache, output gate
        {"name": "attn_tokens_64_fp8", "kind": "attn", "requests": 64, "cached": "256,8192", "new": "1,1",
         "lens_seed": 2, "hq": 16, "hkv": 4, "d": 128, "page": 64, "fp8": True, "gated": True},
        # suffixes (one question each) packed behind long cached prefixes, bf16 cache, output gate
        {"name": "attn_suffixes", "kind": "attn", "requests": 6, "cached": "2048,8192", "new": "30,400",
         "lens_seed": 3, "hq": 16, "hkv": 4, "d": 128, "page": 16, "fp8": False, "gated": True},
        # the last piece of a long prompt fed in pieces, 8/2 heads of 256, 8-bit cache
        {"name": "attn_piece_d256_fp8", "kind": "attn", "requests": 1, "cached": "6144,6144", "new": "2048,2048",
         "lens_seed": 4, "hq": 8, "hkv": 2, "d": 256, "page": 128, "fp8": True, "gated": False},
        # one token each of 64 requests into bf16 pages
        {"name": "write_tokens_64", "kind": "write", "requests": 64, "cached": "256,8192", "new": "1,1", "lens_seed": 5,
         "hkv": 4, "d": 128, "page": 16, "fp8": False},
        # whole prompts packed into one row, quantised as they are written
        {"name": "write_prompts_fp8", "kind": "write", "requests": 4, "cached": "1,1000", "new": "256,8192",
         "lens_seed": 6, "hkv": 4, "d": 128, "page": 64, "fp8": True},
        # a short bf16 prefix read back
        {"name": "read_short", "kind": "read", "requests": 1, "cached": "611,611", "new": "0,0", "lens_seed": 7,
         "hkv": 2, "d": 256, "page": 16, "fp8": False},
        # long prefixes read back from the 8-bit cache
        {"name": "read_prompts_fp8", "kind": "read", "requests": 6, "cached": "256,8192", "new": "0,0", "lens_seed": 8,
         "hkv": 4, "d": 128, "page": 64, "fp8": True},
        # one token of one request through a linear layer's delta rule: latency only
        {"name": "delta_token", "kind": "delta", "requests": 1, "new": "1,1", "lens_seed": 9, "hk": 16, "hv": 16,
         "beta32": False},
        # a decoding step of 64 requests
        {"name": "delta_tokens_64", "kind": "delta", "requests": 64, "new": "1,1", "lens_seed": 10, "hk": 16, "hv": 16,
         "beta32": False},
        # one token each of 64 requests through the conv
        {"name": "conv_tokens_64", "kind": "conv", "requests": 64, "new": "1,1", "lens_seed": 11},
        # suffixes packed into one row, each continued from its own state
        {"name": "conv_suffixes", "kind": "conv", "requests": 12, "new": "30,1500", "lens_seed": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "write", "read", "delta", "conv"])
    seed = rng.randint(1, 1 << 30)
    if kind == "delta":
        tokens = rng.choice([1, 1, rng.randint(2, 12)])
        hk, hv = rng.choice([(16, 16), (16, 16), (8, 16), (4, 8)])
        return {"kind": "delta", "requests": _log_int(rng, 1, 64), "new": f"1,{tokens}", "lens_seed": seed, "hk": hk,
                "hv": hv, "beta32": rng.random() < 0.3}
    if kind == "conv":
        top = rng.choice([1, _log_int(rng, 2, 1500)])
        return {"kind": "conv", "requests": _log_int(rng, 1, 64 if top < 100 else 12), "new": f"1,{top}",
                "lens_seed": seed}
    hq, hkv, d = rng.choice([(16, 4, 128), (16, 4, 128), (8, 2, 256), (16, 4, 64), (8, 8, 128), (6, 1, 128)])
    case = {"kind": kind, "lens_seed": seed, "hkv": hkv, "d": d, "page": rng.choice([16, 16, 32, 64, 128, 256]),
            "fp8": rng.random() < 0.5}
    if kind != "attn":
        top = _log_int(rng, 2, 8192)
        case["requests"] = _log_int(rng, 1, max(1, min(64, 16000 // top)))
        if kind == "read":
            return {**case, "cached": f"1,{top}", "new": "0,0"}
        return {**case, "cached": f"1,{_log_int(rng, 2, 2000)}", "new": f"1,{top}"}
    case |= {"hq": hq, "gated": rng.random() < 0.5}
    top = _log_int(rng, 16, 8192)
    if rng.random() < 0.4:  # single tokens
        return {**case, "requests": _log_int(rng, 1, 64), "cached": f"1,{top}", "new": "1,1"}
    new = _log_int(rng, 2, 1200)
    return {**case, "requests": rng.randint(1, 8 if new <= 100 else 4 if new <= 300 else 1), "cached": f"1,{top}", "new": f"1,{new}"}


# ---------------------------------------------------------------- sizes

def _lens(case):
    """(cached tokens, new tokens) of every request: log-uniform between the case's bounds."""
    rng = random.Random(case["lens_seed"])

    def some(bounds):
        lo, hi = (int(b) for b in bounds.split(","))
        return [lo if lo == hi else _log_int(rng, lo, hi) for _ in range(case["requests"])]
    return some(case.get("cached", "0,0")), some(case["new"])


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def work(case):
    cached, new = _lens(case)
    total, n = sum(new), len(new)
    if case["kind"] == "delta":
        hk, hv = case["hk"], case["hv"]
        rows = total * (2 * hk + 2 * hv) * HEAD * 2 + total * hv * (4 + (4 if case["beta32"] else 2))
        return {"bytes": rows + 2 * n * hv * HEAD * HEAD * 4, "flops": 7 * total * hv * HEAD * HEAD}
    if case["kind"] == "conv":
        c = 3 * 16 * HEAD
        return {"bytes": 2 * (2 * total * c + c * WIDTH + 2 * n * (WIDTH - 1) * c), "flops": 2 * total * c * WIDTH}
    hkv, d = case["hkv"], case["d"]
    held = hkv * (d + 1 if case["fp8"] else 2 * d)  # K or V of one token in the cache
    if case["kind"] == "write":
        return {"bytes": 2 * total * (hkv * d * 2 + held), "flops": 4 * total * hkv * d}
    if case["kind"] == "read":
        return {"bytes": 2 * sum(cached) * (hkv * d * 2 + held), "flops": 2 * sum(cached) * hkv * d}
    pairs = sum(m * c + m * (m + 1) // 2 for c, m in zip(cached, new))
    keys = sum(cached) + total
    return {"bytes": 2 * keys * held + total * case["hq"] * d * 2 * (3 if case["gated"] else 2),
            "flops": 4 * case["hq"] * d * pairs}


# ---------------------------------------------------------------- inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _pages(case, held, gen):
    """A pool a quarter larger than the requests need, its pages dealt to them in random order:
    (pool size, page table [requests, most pages + 1] with -1 where a request has no page)."""
    need = [-(-t // case["page"]) for t in held]
    pool = sum(need) + sum(need) // 4 + 1
    order = torch.randperm(pool, generator=gen, device=DEV).tolist()
    at = _starts(need)
    table = [order[a:b] + [-1] * (max(need) + 1 - (b - a)) for a, b in zip(at, at[1:])]
    return pool, _ints(table)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = _lens(case)
    n, total = len(new), sum(new)
    packed = max(new) != min(new) or case["kind"] == "read"
    s = {"case": case, "new": new, "max_new": max(new), "cu": _ints(_starts(new)) if packed else None}
    if case["kind"] == "delta":
        hk, hv = case["hk"], case["hv"]
        rows = (1, total) if packed else (n, new[0])
        s |= {"q": _normal(gen, *rows, hk, HEAD), "k": _normal(gen, *rows, hk, HEAD), "v": _normal(gen, *rows, hv, HEAD),
              "g": -torch.exp(torch.empty((*rows, hv), device=DEV).uniform_(-4.0, 0.5, generator=gen)),
              "beta": torch.rand((*rows, hv), generator=gen, device=DEV).to(torch.float32 if case["beta32"] else torch.bfloat16),
              "state": _normal(gen, n, hv, HEAD, HEAD, std=0.1, dtype=torch.float32)}
        return s
    if case["kind"] == "conv":
        c = 3 * 16 * HEAD
        rows = (1, total) if packed else (n, new[0])
        s |= {"x": _normal(gen, *rows, c), "w": _normal(gen, c, WIDTH, std=0.3),
              "state": _normal(gen, n, WIDTH - 1, c)}
        s["state_out"] = torch.zeros_like(s["state"])
        return s
    hkv, d, page = case["hkv"], case["d"], case["page"]
    held = [a + b for a, b in zip(cached, new)]
    pool, s["table"] = _pages(case, held, gen)
    s["lens"] = _ints(held)
    shape = (pool, hkv, page, d)
    if case["kind"] == "write":
        kind = torch.float8_e4m3fn if case["fp8"] else torch.bfloat16
        s["kc"], s["vc"] = (torch.zeros(shape, dtype=kind, device=DEV) for _ in range(2))
        s["ks"], s["vs"] = ((torch.full(shape[:3], 127, dtype=torch.uint8, device=DEV) for _ in range(2))
                            if case["fp8"] else (None, None))
        rows = (1, total) if packed else (n, new[0])
        # projections as the layer makes them: [B, T, H, D], read as [B, H, T, D]; rows of unequal size
        s["k"], s["v"] = ((_normal(gen, *rows, hkv, d) * torch.exp2(torch.randint(-2, 3, (*rows, hkv, 1), generator=gen,
                                                                                  device=DEV)).to(torch.bfloat16)).transpose(1, 2)
                          for _ in range(2))
        return s
    if case["fp8"]:
        # rows as the quantiser leaves them: the largest code of each lies between half the range and its end
        s["ks"], s["vs"] = (torch.randint(118, 122, shape[:3], generator=gen, device=DEV, dtype=torch.uint8) for _ in range(2))
        s["kc"], s["vc"] = (_normal(gen, *shape, std=100.0, dtype=torch.float32).clamp_(-E4M3_MAX, E4M3_MAX)
                            .to(torch.float8_e4m3fn) for _ in range(2))
    else:
        s["ks"] = s["vs"] = None
        s["kc"], s["vc"] = (_normal(gen, *shape) for _ in range(2))
    if case["kind"] == "read":
        s["cu"], s["total"] = _ints(_starts(held)), sum(held)
        s["held"] = held
        return s
    hq = case["hq"]
    rows = (1, total) if packed else (n, new[0])
    s["q"] = _normal(gen, *rows, hq, d, std=1.5).transpose(1, 2)
    s["gate"] = _normal(gen, *rows, hq, d).transpose(1, 2) if case["gated"] else None
    s["max_held"] = max(held)
    return s


# ---------------------------------------------------------------- this package's entry points

def _run_own(s):
    kind = s["case"]["kind"]
    if kind == "attn":
        from fastdecisions_amd.paged_gqa_kernel import paged_gqa_attention
        packed = {} if s["cu"] is None else {"cu_seqlens": s["cu"], "max_seqlen": s["max_new"]}
        return paged_gqa_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], k_scale=s["ks"], v_scale=s["vs"],
                                   gate=s["gate"], **packed)
    if kind == "write":
        from fastdecisions_amd.paged_kv_kernel import paged_kv_write
        paged_kv_write(s["k"], s["v"], s["kc"], s["vc"], s["table"], s["lens"], k_scale=s["ks"], v_scale=s["vs"],
                       cu_seqlens=s["cu"])
        return [s["kc"], s["vc"], s["ks"], s["vs"]]
    if kind == "read":
        from fastdecisions_amd.paged_kv_kernel import paged_kv_read
        return list(paged_kv_read(s["kc"], s["vc"], s["table"], s["cu"], s["total"], k_scale=s["ks"], v_scale=s["vs"]))
    if kind == "delta":
        from fastdecisions_amd.gated_delta_kernel import recurrent_gated_delta_rule
        return list(recurrent_gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["state"],
                                               output_final_state=True, use_qk_l2norm_in_kernel=True,
                                               cu_seqlens=s["cu"]))
    from fastdecisions_amd.packed_conv_kernel import prep_qkv_state
    out = prep_qkv_state(s["x"], s["w"], s["state"], cu_seqlens=s["cu"], state_out=s["state_out"])
    return [*out, s["state_out"]]


# ---------------------------------------------------------------- plain forms

def _where(s):
    """(request, index within it) of every new token in packed order."""
    new = torch.tensor(s["new"], device=DEV)
    req = torch.repeat_interleave(torch.arange(len(s["new"]), device=DEV), new)
    first = torch.cumsum(new, 0) - new
    return req, torch.arange(req.numel(), device=DEV) - first[req]


def _dense(s, cache, scale, length):
    """The first `length` keys of every request [requests, heads, length, d] in 32 bits."""
    page = s["case"]["page"]
    table = s["table"][:, :-(-length // page)].long().clamp(min=0)
    x = cache.view(torch.uint8)[table].view(cache.dtype).float() if scale is not None else cache[table].float()
    if scale is not None:
        x = x * (scale[table].to(torch.int32) << 23).view(torch.float32)[..., None]  # 2^(byte - 127)
    n, p, h, _, d = x.shape
    return x.transpose(1, 2).reshape(n, h, p * page, d)[:, :, :length]


def _plain_attn(s):
    q, lens = s["q"], s["lens"].long()
    n, new, length = lens.numel(), s["max_new"], s["max_held"]
    hq, d = q.shape[1], q.shape[3]
    hkv = s["kc"].shape[1]
    if s["cu"] is None:
        qd = q.float()
    else:
        req, at = _where(s)
        qd = torch.zeros((n, hq, new, d), device=DEV)
        qd[req, :, at] = q[0].transpose(0, 1).float()
    k, v = _dense(s, s["kc"], s["ks"], length), _dense(s, s["vc"], s["vs"], length)
    count = torch.tensor(s["new"], device=DEV)
    last = (lens - count)[:, None] + torch.arange(new, device=DEV)      # position of each new token
    keys = torch.arange(length, device=DEV)
    v = torch.where((keys < lens[:, None])[:, None, :, None], v, 0.0)   # what lies behind a request never counts
    seen = keys <= torch.minimum(last, lens[:, None] - 1)[..., None]    # [requests, new, length]
    p = qd.reshape(n, hkv, -1, d) @ k.transpose(2, 3)
    p = (p * d ** -0.5).reshape(n, hq, new, length).masked_fill_(~seen[:, None], float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(n, hkv, -1, length) @ v).reshape(n, hq, new, d) / total
    if s["cu"] is not None:
        o = o[req, :, at].transpose(0, 1)[None]
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(torch.bfloat16)


def _plain_write(s):
    page = s["case"]["page"]
    req, at = _where(s)
    count = torch.tensor(s["new"], device=DEV)
    pos = (s["lens"].long() - count)[req] + at
    slot = s["table"].long()[req, pos // page]
    for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])       # [tokens, heads, d]
        if scale is None:
            cache[slot, :, pos % page] = x
            continue
        x = x.float()
        top = x.abs().amax(-1)
        m, e = torch.frexp(top / torch.full_like(top, E4M3_MAX))        # top / 448 = m 2^e, m in [0.5, 1)
        e = torch.where(top > 0, torch.where(m > 0.5, e, e - 1), 0).clamp(min=-126).to(torch.int32)
        code = (x * ((127 - e) << 23).view(torch.float32)[..., None]).to(torch.float8_e4m3fn)  # 2^-e, exactly
        cache.view(torch.uint8)[slot, :, pos % page] = code.view(torch.uint8)
        scale[slot, :, pos % page] = (e + 127).to(torch.uint8)
    return [s["kc"], s["vc"], s["ks"], s["vs"]]


def _plain_read(s):
    held = torch.tensor(s["held"], device=DEV)
    req = torch.repeat_interleave(torch.arange(held.numel(), device=DEV), held)
    at = torch.arange(s["total"], device=DEV) - (torch.cumsum(held, 0) - held)[req]
    out = []
    for cache, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        x = _dense(s, cache, scale, max(s["held"]))[req, :, at]          # [total, heads, d]
        out.append(x.to(torch.bfloat16).transpose(0, 1)[None])
    return out


def _plain_delta(s):
    case, n, new = s["case"], len(s["new"]), s["max_new"]
    hk, hv = case["hk"], case["hv"]
    x = {name: s[name].float() for name in ("q", "k", "v", "g", "beta")}
    for name in ("q", "k"):
        x[name] = x[name] / torch.sqrt((x[name] * x[name]).sum(-1, keepdim=True) + 1e-6)
        x[name] = x[name].repeat_interleave(hv // hk, dim=2)
    if s["cu"] is not None:  # to a padded batch: a row that is not there neither decays nor adds
        req, at = _where(s)
        for name, t in x.items():
            pad = torch.zeros((n, new, *t.shape[2:]), device=DEV)
            pad[req, at] = t[0]
            x[name] = pad
    state, outs = s["state"], []
    for t in range(new):
        k, v, q = x["k"][:, t], x["v"][:, t], x["q"][:, t] * HEAD ** -0.5
        state = state * torch.exp(x["g"][:, t])[..., None, None]
        seen = (state * k[..., None]).sum(-2)
        state = state + k[..., None] * (x["beta"][:, t][..., None] * (v - seen))[..., None, :]
        outs.append((state * q[..., None]).sum(-2))
    out = torch.stack(outs, dim=1)
    if s["cu"] is not None:
        out = out[req, at][None]
    return [out.to(torch.bfloat16), state]


def _plain_conv(s):
    n, new, c = len(s["new"]), s["max_new"], s["x"].shape[2]
    req, at = _where(s)
    x = torch.zeros((n, new + WIDTH - 1, c), device=DEV)
    x[:, :WIDTH - 1] = s["state"].float()
    x[req, at + WIDTH - 1] = s["x"].reshape(-1, c).float()
    w = s["w"].float()
    y = x[:, :new] * w[:, 0]
    for j in range(1, WIDTH):
        y += x[:, j:j + new] * w[:, j]
    y = (y / (1.0 + torch.exp(-y)))[req, at].to(torch.bfloat16)
    shape = (*s["x"].shape[:2], 16, HEAD)
    ends = torch.tensor(s["new"], device=DEV)[:, None] + torch.arange(WIDTH - 1, device=DEV)
    s["state_out"].copy_(x[torch.arange(n, device=DEV)[:, None], ends])
    return [*(p.reshape(shape) for p in y.split(c // 3, dim=1)), s["state_out"]]


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "write": _plain_write, "read": _plain_read, "delta": _plain_delta,
            "conv": _plain_conv}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- in 64 bits

def _rows64(s, r, cache, scale, length):
    """Keys 0 .. length - 1 of request r, [heads, length, d]."""
    page = s["case"]["page"]
    at = torch.arange(length, device=DEV)
    pages, within = s["table"][r].long()[at // page], at % page
    x = cache.double()[pages, :, within]
    if scale is not None:
        x = x * _pow2(scale[pages, :, within].to(torch.int64) - 127)[..., None]
    return x.permute(1, 0, 2)


def _pow2(e):
    """2^e in 64 bits, exactly (a library's pow need not be)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_e4m3(x):
    """(codes' values, scale bytes) of rows x [.., d]."""
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp(min=1e-300) / torch.full_like(top, E4M3_MAX))), 0.0).clamp(min=-126)
    y = x / _pow2(e)[..., None]
    step = _pow2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, (e + 127).to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    kind, starts = case["kind"], _starts(s["new"])
    count = len(s["new"])
    if kind == "attn":
        hq, d, hkv = case["hq"], case["d"], case["hkv"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for r, m in enumerate(s["new"]):
            row, a = (r, 0) if s["cu"] is None else (0, starts[r])
            length = int(s["lens"][r])
            k, v = _rows64(s, r, s["kc"], s["ks"], length), _rows64(s, r, s["vc"], s["vs"], length)
            for h in range(hq):
                z = s["q"][row, h, a:a + m].double() @ k[h * hkv // hq].T / math.sqrt(d)
                z += torch.full_like(z, -math.inf).triu(length - m + 1)
                o = torch.softmax(z, dim=-1) @ v[h * hkv // hq]
                if s["gate"] is not None:
                    o *= torch.sigmoid(s["gate"][row, h, a:a + m].double())
                out[row, h, a:a + m] = o
        return out
    if kind == "write":
        res = []
        for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
            values = cache.double()
            scales = None if scale is None else scale.clone()
            for r, m in enumerate(s["new"]):
                row, a = (r, 0) if s["cu"] is None else (0, starts[r])
                pos = int(s["lens"][r]) - m + torch.arange(m, device=DEV)
                pages, within = s["table"][r].long()[pos // case["page"]], pos % case["page"]
                y = x[row, :, a:a + m].double().transpose(0, 1)
                if scales is not None:
                    y, scales[pages, :, within] = _exact_e4m3(y)
                values[pages, :, within] = y
            res.append((values, scales))
        (k, ks), (v, vs) = res
        return [k, v, ks, vs]
    if kind == "read":
        return [torch.cat([_rows64(s, r, c, e, m) for r, m in enumerate(s["held"])], dim=1)[None]
                for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]
    if kind == "delta":
        group = case["hv"] // case["hk"]
        out = torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV)
        states = s["state"].double()
        for r, m in enumerate(s["new"]):
            row, a = (r, 0) if s["cu"] is None else (0, starts[r])
            for t in range(a, a + m):
                k, q = (torch.repeat_interleave(x / torch.sqrt((x ** 2).sum(-1, keepdim=True) + 1e-6), group, dim=0)
                        for x in (s["k"][row, t].double(), s["q"][row, t].double()))
                st = states[r] * torch.exp(s["g"][row, t].double())[:, None, None]
                d = s["beta"][row, t].double()[:, None] * (s["v"][row, t].double() - torch.einsum("hij,hi->hj", st, k))
                states[r] = st + torch.einsum("hi,hj->hij", k, d)
                out[row, t] = torch.einsum("hij,hi->hj", states[r], q) / math.sqrt(HEAD)
        return [out, states]
    c = s["x"].shape[2]
    w = s["w"].double()
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device=DEV)
    state = torch.zeros(s["state"].shape, dtype=torch.float64, device=DEV)
    for r in range(count):
        row, a, b = (r, 0, s["new"][r]) if s["cu"] is None else (0, starts[r], starts[r + 1])
        x = torch.cat([s["state"][r], s["x"][row, a:b]]).double()
        z = sum(x[j:j + b - a] * w[:, j] for j in range(WIDTH))
        y[row, a:b] = z * torch.sigmoid(z)
        state[r] = x[-(WIDTH - 1):]
    return [*(p.reshape(*p.shape[:2], 16, HEAD) for p in y.split(c // 3, dim=2)), state]
