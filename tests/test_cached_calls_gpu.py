"""Cached forwards under torch.compile's tracing, and the op of the chunked delta rule between states."""
from __future__ import annotations

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("new", [2, 40])
def test_a_cached_step_traces_whole(new):
    """A token step and a prompt piece (the two forms of the delta rule) are graphs without a break; the traced
    calls are the eager ones, bit for bit."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels, synthetic_ids
    announce(f"traced cached step of {new} tokens")
    model = build_decider(TINY, seed=3)
    install_hip_kernels(model)
    ids = synthetic_ids(1, 2 * new, TINY.vocab_size, seed=1)
    torch._dynamo.reset()
    traced = torch.compile(lambda i, step: model(i, cache=step), backend="eager", fullgraph=True)
    out = []
    for call in (lambda i, step: model(i, cache=step), traced):
        cache = DeciderCache(TINY, requests=1, tokens=200)
        slot = cache.open()
        out.append([call(part, cache.step([slot], [new])) for part in (ids[:, :new], ids[:, new:])])
    for eager, got in zip(*out):
        assert torch.equal(eager, got)


@torch.no_grad()
def test_the_op_of_the_rule_between_states():
    import fastdecisions_amd.cached_ops as ops
    announce("opcheck of gated_delta_rule_states")
    r = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 3, 3, 70], dtype=torch.int32, device="cuda")
    g, beta = -torch.rand((1, 70, 16), device="cuda"), torch.rand((1, 70, 16), device="cuda").to(torch.bfloat16)
    torch.library.opcheck(ops.gated_delta_rule_states_op,
                          (r(1, 70, 16, 128), r(1, 70, 16, 128), r(1, 70, 16, 128), g, beta,
                           torch.randn((3, 16, 128, 128), device="cuda"), cu),
                          test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))
