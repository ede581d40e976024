"""4-bit paged caches for the tests: pools, their rows in 64 bits, and the rule by which rows are held."""
from __future__ import annotations

import torch

from cache_reference import make_pages, pow2

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = 32


def pack(code):
    """Codes [.., d] (uint8, one a byte) as a float4_e2m1fn_x2 pool [.., d / 2]."""
    return (code[..., ::2] | (code[..., 1::2] << 4)).contiguous().view(torch.float4_e2m1fn_x2)


def codes(pool):
    byte = pool.view(torch.uint8)
    return torch.stack([byte & 15, byte >> 4], dim=-1).flatten(-2)


def values(pool, scale):
    """What a pool's rows stand for, in float64."""
    code = codes(pool).long()
    v = torch.tensor(VALUES, dtype=torch.float64, device=pool.device)[code & 7]
    v = torch.where(code >= 8, -v, v).unflatten(-1, (-1, BLOCK))
    s = torch.where(scale == 255, torch.nan, pow2(scale.long()))
    return (v * s[..., None]).flatten(-2)


def hold(x):
    """(codes, scale bytes) of float64 rows x [.., d], value by value: per block the smallest 2^E (E >= -126) with
    max|x| <= 6 2^E over its finite values, codes to nearest even; 2^128 and more is no bf16 number."""
    x = x.unflatten(-1, (-1, BLOCK))
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    _, e = torch.frexp(top)                        # top = m 2^e, m in [0.5, 1); 6 = 0.75 2^3
    e = e.to(torch.int64) - 3
    e = torch.where(top > 6.0 * pow2(e + 127), e + 1, e)
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-126)
    y = (x / pow2(e + 127)[..., None]).abs()
    y = torch.minimum(y, torch.where(e == 126, 3.0, 6.0)[..., None])
    v = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    away = (torch.nan_to_num(y)[..., None] - v).abs()
    near = away == away.amin(-1, keepdim=True)     # two codes on a tie: the even one
    code = torch.where(near, torch.arange(8, device=x.device) + 8 * (torch.arange(8, device=x.device) % 2), 99).amin(-1) % 8
    code = code | (torch.signbit(x).long() << 3)
    scale = torch.where(torch.isnan(x).any(-1), 255, e + 127)
    return code.flatten(-2).to(torch.uint8), scale.to(torch.uint8)


def make_pages4(lens, page, heads, dim, seed, **kw):
    """As ``make_pages``: pages of N(0, 1) rows held in 4 bits, features of unequal size."""
    c = make_pages(lens, page, heads, dim, False, seed, **kw)
    gen = torch.Generator(device=c["k"].device).manual_seed(seed + 1)
    for name in ("k", "v"):
        x = c[name].double()
        x = x * pow2(torch.randint(125, 129, (*x.shape[:3], dim // 16), generator=gen, device=x.device)).repeat_interleave(16, -1)
        code, scale = hold(x)
        c[name], c[name + "s"] = pack(code), scale
    return c


def rows4(c, name, r, n):
    """``cache_reference.rows`` of a 4-bit cache."""
    pool, page = c[name].shape[0], c["page"]
    at = torch.arange(n, device=c["table"].device)
    pages = c["table"][r].long()[at // page]
    there = (pages >= 0) & (pages < pool)
    pages = pages.clamp(0, pool - 1)
    x = values(c[name].view(torch.uint8)[pages, :, at % page].view(torch.float4_e2m1fn_x2), c[name + "s"][pages, :, at % page])
    return x.permute(1, 0, 2), there
