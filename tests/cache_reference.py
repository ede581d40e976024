"""Paged caches for the tests and the cache operators in 64 bits, one request and head at a time."""
from __future__ import annotations

import math

import torch

HALF_STEP = 2.0 ** -8  # half a bf16 step, relative


def make_pages(lens, page, heads, dim, fp8, seed, extra_pages=3, spare_entries=1, device="cuda"):
    """A pool whose pages hold N(0, 1) rows, dealt to the requests in random order: dict of k, v, ks, vs
    and table (its spare entries -1)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pool = sum(need) + extra_pages
    order = torch.randperm(pool, generator=gen, device=device).tolist()
    table = torch.full((len(lens), max(need + [1]) + spare_entries), -1, dtype=torch.int32)
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    k, v = (torch.randn((pool, heads, page, dim), generator=gen, device=device) for _ in range(2))
    c = {"table": table.to(device), "ks": None, "vs": None, "page": page, "device": device}
    if fp8:
        for name, x in (("k", k), ("v", v)):
            c[name + "s"] = torch.randint(119, 122, x.shape[:3], generator=gen, device=device, dtype=torch.uint8)
            c[name] = (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        c["k"], c["v"] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    return c


def pow2(byte):
    """2^(byte - 127) in float64, exactly."""
    return ((byte.to(torch.int64) - 127 + 1023) << 52).view(torch.float64)


def rows(c, name, r, n):
    """(keys or values 0 .. n - 1 of request r [heads, n, dim] in float64, which of them lie on a page)."""
    pool, page = c[name].shape[0], c["page"]
    at = torch.arange(n, device=c[name].device)
    pages = c["table"][r].long()[at // page]
    there = (pages >= 0) & (pages < pool)
    x = c[name].to(torch.float64)[pages.clamp(0, pool - 1), :, at % page]
    if c[name + "s"] is not None:
        x = x * pow2(c[name + "s"][pages.clamp(0, pool - 1), :, at % page])[..., None]
    return x.permute(1, 0, 2), there


def attention(q, c, length, scale, gate=None):
    """Attention of the n last tokens of a request of `length` keys, q [Hq, n, D], in float64: (out, bound).
    c: (k, v, there) of the request, [Hkv, length, D] each.

    The bound on |kernel - out|: probabilities are rounded to bf16 in the product and, as rounded, in the
    denominator (half a step each, against sum p |v|), the result once; 2^-12 covers the fp32 scores, exp2 and
    sums (a score of |s| < 64 in fp32 over 256 products is off by less than 2^-14)."""
    k, v, there = c
    hq, n, dim = q.shape
    group = hq // k.shape[0]
    out = torch.zeros((hq, n, dim), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    if length > 0 and n > 0:
        pos = length - n + torch.arange(n, device=q.device)
        keys = torch.arange(length, device=q.device)
        seen = (keys[None, :] <= pos[:, None]) & there[None, :]
        for h in range(hq):
            kh, vh = k[h // group], v[h // group]
            s = torch.where(seen, (q[h].double() @ kh.T) * scale, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            out[h] = p @ vh
            mag[h] = p @ vh.abs()
    if gate is not None:
        sig = torch.sigmoid(gate.double())
        out, mag = out * sig, mag * sig
    return out, (2 * HALF_STEP + 2.0 ** -12) * mag * (1 + 2.0 ** -7) + HALF_STEP * out.abs() + 1e-30


def e4m3(x):
    """(codes' values, scale bytes) of float64 rows x [.., d]: the rule of fd_paged_kv_write, value by value."""
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
    top = finite.amax(-1)
    _, e = torch.frexp(top)                      # top = m 2^e, m in [0.5, 1)
    e = e.to(torch.int64) - 9                    # 448 = 0.875 2^9
    e = torch.where(top > 448.0 * pow2(e + 127), e + 1, e)
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-126)
    y = (x / pow2(e + 127)[..., None]).clamp(-448, 448)
    _, ey = torch.frexp(torch.where(torch.isnan(y), 1.0, y).abs().clamp(min=2.0 ** -6))
    step = pow2(ey.to(torch.int64) - 1 - 3 + 127)
    return torch.round(y / step) * step, (e + 127).to(torch.uint8)
