"""The delta rule token by token and the conv continued from a state, on the GPU."""
from __future__ import annotations

import pytest
import torch

from cache_reference import HALF_STEP
from helpers import announce

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------- the delta rule

def delta_inputs(rows, hk, hv, seed, beta_dtype=torch.bfloat16, unit=False):
    g_ = gen(seed)
    q, k = (torch.randn((*rows, hk, 128), generator=g_, device="cuda") for _ in range(2))
    if unit:
        q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    v = torch.randn((*rows, hv, 128), generator=g_, device="cuda").to(torch.bfloat16)
    g = -torch.exp(torch.empty((*rows, hv), device="cuda").uniform_(-4.0, 1.0, generator=g_))
    beta = torch.rand((*rows, hv), generator=g_, device="cuda").to(beta_dtype)
    return q.to(torch.bfloat16), k.to(torch.bfloat16), v, g, beta


def delta_reference(q, k, v, g, beta, state, norm, scale=128 ** -0.5):
    """One request, rows [n, H, 128], state [Hv, 128, 128], in float64: (out, state, bounds of both).

    Every step of the kernel rounds in fp32: products over 128 rows, the decay and the update, under 140
    roundings against the columns' norm and |v|.  With |k| <= 1 and beta <= 1 a step does not enlarge an
    error of its state (|I - beta k k^T| <= 1, e^g <= 1), so errors add up over the steps."""
    n, hv = v.shape[0], v.shape[1]
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if norm:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q, k = (x.repeat_interleave(hv // x.shape[1], dim=1) for x in (q, k))
    s = state.double().clone()
    out, bound = torch.zeros_like(v), torch.zeros_like(v)
    off = torch.zeros((hv, 128), dtype=torch.float64, device=v.device)  # of each column, 2-norm
    eps = 140 * 2.0 ** -24
    for t in range(n):
        size = s.norm(dim=1)
        s = s * torch.exp(g[t])[:, None, None]
        d = beta[t][:, None] * (v[t] - (s * k[t][..., None]).sum(1))
        s = s + k[t][..., None] * d[:, None, :]
        off = off + eps * (size + v[t].abs())
        out[t] = (s * q[t][..., None]).sum(1) * scale
        reach = q[t].norm(dim=-1)[:, None] * scale
        bound[t] = reach * (off + eps * (size + v[t].abs())) + HALF_STEP * out[t].abs() + 1e-30
    return out, s, bound, off[:, None, :] + 1e-30


def check_delta(q, k, v, g, beta, state, out, final, new, packed, norm, scale=128 ** -0.5):
    at = starts(new)
    for r, n in enumerate(new):
        take = (lambda t: t[0, at[r]:at[r + 1]]) if packed else (lambda t: t[r])
        want, s, bound, s_bound = delta_reference(*(take(x) for x in (q, k, v, g, beta)), state[r], norm, scale)
        assert ((take(out).double() - want).abs() <= bound).all(), f"request {r}: out"
        if final is not None:
            assert ((final[r].double() - s).abs() <= s_bound).all(), f"request {r}: state"


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("beta_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hk,hv,B,T", [(16, 16, 1, 1), (8, 16, 3, 1), (4, 8, 5, 7), (1, 3, 2, 33)])
def test_tokens(hk, hv, B, T, beta_dtype, norm):
    from fastdecisions_amd.gated_delta_kernel import recurrent_gated_delta_rule
    announce(f"delta step B={B} T={T} {hk}/{hv} heads, beta {beta_dtype}, norm {norm}")
    x = delta_inputs((B, T), hk, hv, 30 + T, beta_dtype, unit=not norm)
    state = torch.randn((B, hv, 128, 128), generator=gen(1), device="cuda") * 0.3
    keep = state.clone()
    out, final = recurrent_gated_delta_rule(*x, initial_state=state, output_final_state=True, use_qk_l2norm_in_kernel=norm)
    assert torch.equal(state, keep)
    check_delta(*x, state, out, final, [T] * B, False, norm)
    out2, none = recurrent_gated_delta_rule(*x, initial_state=state, use_qk_l2norm_in_kernel=norm)
    assert none is None and torch.equal(out, out2)
    out0, final0 = recurrent_gated_delta_rule(*x, output_final_state=True, use_qk_l2norm_in_kernel=norm, scale=0.3)
    check_delta(*x, torch.zeros_like(state), out0, final0, [T] * B, False, norm, scale=0.3)


def test_packed_requests():
    """Requests of unequal length, empty ones among them (whose state is handed on), rows behind the last."""
    from fastdecisions_amd.gated_delta_kernel import recurrent_gated_delta_rule
    announce("delta step, packed")
    new = [3, 0, 1, 20, 0, 1]
    x = delta_inputs((1, sum(new) + 4), 4, 8, 31)
    state = torch.randn((len(new), 8, 128, 128), generator=gen(2), device="cuda") * 0.3
    out, final = recurrent_gated_delta_rule(*x, initial_state=state, output_final_state=True,
                                            use_qk_l2norm_in_kernel=True, cu_seqlens=ints(starts(new)))
    check_delta(*x, state, out, final, new, True, True)
    assert torch.equal(final[1], state[1]) and torch.equal(final[4], state[4])


def test_rows_behind_the_last_request_stay():
    from fastdecisions_amd import _cache_lib, _lib
    announce("delta step and conv, rows behind the last request")
    q, k, v, g, beta = delta_inputs((1, 9), 2, 2, 32)
    out = torch.full_like(v, 5.0)
    state = torch.zeros((2, 2, 128, 128), device="cuda")
    cu = ints([0, 2, 6])
    _cache_lib.check("fd_gated_delta_step", _cache_lib.lib().fd_gated_delta_step(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(), state.data_ptr(), None,
        2, None, 1, 9, 2, 2, 128, 128, 1.0, 0, 1, cu.data_ptr(), 2, _lib.stream_handle(q.device)))
    assert (out[0, 6:] == 5.0).all() and (out[0, :6] != 5.0).any()
    x, w = conv_inputs((1, 9), 384, 4, 33)
    qkv = [torch.full((1, 9, 128), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    conv = torch.zeros((2, 3, 384), dtype=torch.bfloat16, device="cuda")
    _cache_lib.check("fd_packed_conv_state", _cache_lib.lib().fd_packed_conv_state(
        x.data_ptr(), 384, w.data_ptr(), None, conv.data_ptr(), conv.data_ptr(), 2, None, *(t.data_ptr() for t in qkv),
        1, 9, 128, 128, 4, cu.data_ptr(), 2, 1, _lib.stream_handle(q.device)))
    assert all((t[0, 6:] == 5.0).all() and (t[0, :6] != 5.0).all() for t in qkv)


def test_state_pool():
    """States in a pool: rows of other requests untouched, indices out of range and repeated ones no state."""
    from fastdecisions_amd.gated_delta_kernel import recurrent_gated_delta_rule
    announce("delta step, state pool")
    n = 70  # more requests than lanes
    x = delta_inputs((n, 2), 1, 2, 34)
    pool = torch.randn((100, 2, 128, 128), generator=gen(3), device="cuda") * 0.3
    order = torch.randperm(100, generator=torch.Generator().manual_seed(4))[:n].tolist()
    order[5], order[6], order[69], order[66] = -1, 100, order[2], order[2]
    before = pool.clone()
    out, same = recurrent_gated_delta_rule(*x, initial_state=pool, use_qk_l2norm_in_kernel=True, state_indices=ints(order))
    assert same is pool
    lost = [5, 6, 66, 69]
    state = torch.stack([torch.zeros_like(pool[0]) if r in lost else before[order[r]] for r in range(n)])
    final = torch.stack([state[r] if r in lost else pool[order[r]] for r in range(n)])
    keep = [r for r in range(n) if r not in lost]
    check_delta(*x, state, out, None, [2] * n, False, True)
    check_delta(*(t[keep] for t in x), state[keep], out[keep], final[keep], [2] * len(keep), False, True)
    others = [i for i in range(100) if i not in {order[r] for r in keep}]
    assert torch.equal(pool[others], before[others])
    # written to another pool at the same rows
    other = torch.zeros_like(pool)
    out2, _ = recurrent_gated_delta_rule(*x, initial_state=before, use_qk_l2norm_in_kernel=True,
                                         state_indices=ints(order), state_out=other)
    assert torch.equal(out, out2) and torch.equal(other[[order[r] for r in keep]], pool[[order[r] for r in keep]])
    assert other[others].abs().max() == 0


def test_tokens_continue_the_chunked_rule():
    """A prompt on the chunked rule, then tokens one by one: the chunked rule over everything.  The two round
    the normalised q and k differently (bf16 there), so outputs agree within those roundings."""
    from fastdecisions_amd.gated_delta_kernel import chunk_gated_delta_rule, recurrent_gated_delta_rule
    announce("delta step after the chunked rule")
    x = delta_inputs((2, 140), 4, 8, 35)
    whole, last = chunk_gated_delta_rule(*x, output_final_state=True, use_qk_l2norm_in_kernel=True)
    _, state = chunk_gated_delta_rule(*(t[:, :130].contiguous() for t in x), output_final_state=True,
                                      use_qk_l2norm_in_kernel=True)
    pool = state.clone()
    outs = [recurrent_gated_delta_rule(*(t[:, i:i + 1].contiguous() for t in x), initial_state=pool, state_out=pool,
                                       use_qk_l2norm_in_kernel=True)[0] for i in range(130, 140)]
    got = torch.cat(outs, dim=1).double()
    want = whole[:, 130:].double()
    # l2norm's bf16 roundings: three a value (square sum, inverse root, product), 2^-8 each, on q and on k
    assert (got - want).norm() <= 6 * HALF_STEP * want.norm()
    assert (pool - last).norm() <= 6 * HALF_STEP * last.norm()


def test_captured_step():
    """A captured step replayed: the pool moves on as eager calls move it, the indices may change between."""
    from fastdecisions_amd.gated_delta_kernel import recurrent_gated_delta_rule
    announce("delta step, captured")
    x = delta_inputs((3, 1), 2, 4, 36)
    pool = torch.randn((6, 4, 128, 128), generator=gen(5), device="cuda") * 0.3
    twin, idx = pool.clone(), ints([0, 1, 2])
    call = lambda p: recurrent_gated_delta_rule(*x, initial_state=p, use_qk_l2norm_in_kernel=True, state_indices=idx)[0]
    call(twin.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(pool)
    for now in ([0, 1, 2], [2, 0, 5], [3, 3, 1]):
        idx.copy_(ints(now))
        for t in x:
            t.copy_(t.roll(1, 0))
        graph.replay()
        want = call(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pool, twin)


# ---------------------------------------------------------------- the conv

def conv_inputs(rows, channels, width, seed):
    g_ = gen(seed)
    x = torch.randn((*rows, channels), generator=g_, device="cuda").to(torch.bfloat16)
    w = (torch.randn((channels, width), generator=g_, device="cuda") * 0.4).to(torch.bfloat16)
    return x, w


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("activation", ["silu", None])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("key_dim,value_dim", [(2048, 2048), (128, 256)])
def test_pieces_are_the_whole(key_dim, value_dim, bias, activation, width):
    """A request fed in pieces from a zero state: the uncached conv's bits, whatever the cuts."""
    from fastdecisions_amd.packed_conv_kernel import prep_qkv, prep_qkv_state
    announce(f"conv state, pieces, {key_dim}/{value_dim}, width {width}, bias {bias}, {activation}")
    channels = 2 * key_dim + value_dim
    x, w = conv_inputs((2, 101), channels, width, 40)
    b = (torch.randn(channels, generator=gen(41), device="cuda") * 0.2).to(torch.bfloat16) if bias else None
    kw = dict(key_dim=key_dim, value_dim=value_dim, activation=activation)
    want = prep_qkv(x, w, b, **kw)
    state = torch.zeros((2, width - 1, channels), dtype=torch.bfloat16, device="cuda")
    done, parts = 0, []
    for n in (1, 2, 1, 3, 40, 8, 1, 1, 16, 28):
        parts.append(prep_qkv_state(x[:, done:done + n].contiguous(), w, state, b, **kw))
        done += n
    assert done == 101
    for i in range(3):
        assert torch.equal(torch.cat([p[i] for p in parts], dim=1).view(torch.int16), want[i].view(torch.int16))
    assert torch.equal(state, x[:, -(width - 1):])


@pytest.mark.parametrize("new", [[1, 0, 2, 50, 3, 1, 4, 17], [9] * 3 + [600], [1] * 90])
def test_packed_suffixes(new):
    """Requests packed into one row of a wider projection, each continued from its state in a pool; rows of
    the pool that no request owns stay; repeated and absent indices are no state."""
    from fastdecisions_amd.packed_conv_kernel import prep_qkv, prep_qkv_state
    announce(f"conv state, packed {len(new)} requests")
    n, total = len(new), sum(new)
    wide, w = conv_inputs((1, total), 512, 4, 42)
    w = w[:384].contiguous()
    x = wide[..., :384]
    pool = torch.randn((n + 3, 3, 384), generator=gen(43), device="cuda").to(torch.bfloat16)
    order = torch.randperm(n + 3, generator=torch.Generator().manual_seed(5))[:n].tolist()
    lost = []
    if n > 4:
        order[n - 1], order[n - 2], lost = order[0], -5, [n - 1, n - 2]
    before = pool.clone()
    out = prep_qkv_state(x, w, pool, cu_seqlens=ints(starts(new)), state_indices=ints(order))
    at = starts(new)
    owned = {}
    for r, m in enumerate(new):
        state = torch.zeros_like(before[0]) if r in lost else before[order[r]]
        full = torch.cat([state, x[0, at[r]:at[r + 1]]])[None].contiguous()
        if m:
            want = prep_qkv(full, w)
            for got, y in zip(out, want):
                assert torch.equal(got[0, at[r]:at[r + 1]].view(torch.int16), y[0, 3:].view(torch.int16)), f"request {r}"
        if r not in lost:
            owned[order[r]] = full[0, -3:]
    for i in range(n + 3):
        assert torch.equal(pool[i], owned.get(i, before[i])), f"state {i}"


def test_state_to_another_tensor():
    from fastdecisions_amd.packed_conv_kernel import prep_qkv_state
    announce("conv state written elsewhere")
    x, w = conv_inputs((3, 2), 384, 4, 44)
    state = torch.randn((3, 3, 384), generator=gen(45), device="cuda").to(torch.bfloat16)
    keep, other = state.clone(), torch.zeros_like(state)
    out = prep_qkv_state(x, w, state, state_out=other)
    assert torch.equal(state, keep) and torch.equal(other, torch.cat([state, x], dim=1)[:, -3:])
    again = prep_qkv_state(x, w, state)  # in place
    assert torch.equal(state, other) and all(torch.equal(a, b) for a, b in zip(out, again))
