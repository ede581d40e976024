"""What a layer's forward over a step of a cache refuses, whichever way it is called (no GPU)."""
from __future__ import annotations

import pytest
import torch

from fastdecisions_amd.decider_cache import DeciderCache
from fastdecisions_amd.model import TINY, build_decider, install_hip_kernels


@pytest.fixture(scope="module")
def layers():
    model = build_decider(TINY, seed=1, device="cpu")
    install_hip_kernels(model)
    linear = next(m.linear_attn for m in model.core.layers if getattr(m, "linear_attn", None) is not None)
    attention = next(m.self_attn for m in model.core.layers if getattr(m, "self_attn", None) is not None)
    return model, linear, attention


def calls(layers, step, x, **kw):
    """One call of each kind of layer over the step."""
    model, linear, attention = layers
    pe = model.core.rotary_emb(x, step.positions)
    return (lambda: linear(x, fd_cache=step, **({"cache_params": kw["cache"]} if "cache" in kw else kw)),
            lambda: attention(x, pe, fd_cache=step, **({"past_key_values": kw["cache"]} if "cache" in kw else kw)))


def make(n=6):
    cache = DeciderCache(TINY, requests=1, tokens=64, device="cpu")
    return cache.step([cache.open()], [n]), torch.zeros((1, n, TINY.hidden_size), dtype=torch.bfloat16)


def test_gradients_are_refused(layers):
    """A result without its gradient is no answer to a call that asks for one."""
    step, x = make()
    with torch.enable_grad():
        for call in calls(layers, step, x):
            with pytest.raises(RuntimeError, match="inference"):
                call()


@torch.no_grad()
def test_dropout_is_refused(layers, monkeypatch):
    step, x = make()
    attention = layers[2]
    monkeypatch.setattr(attention, "attention_dropout", 0.1)
    attention.train()
    try:
        with pytest.raises(RuntimeError, match="eval mode"):
            calls(layers, step, x)[1]()
    finally:
        attention.eval()


@torch.no_grad()
@pytest.mark.parametrize("other", [{"attention_mask": torch.zeros(1, 1, 6, 6)}, {"cache": object()}])
def test_masks_and_other_caches_are_refused(layers, other):
    """They were passed over: the layer computed as if there were none."""
    step, x = make()

    class OnGpu(torch.Tensor):  # the check of the device comes first; nothing is computed
        is_cuda = True
    for call in calls(layers, step, x.as_subclass(OnGpu), **other):
        with pytest.raises(ValueError, match="beside fd_cache"):
            call()


@torch.no_grad()
def test_other_devices_and_types_are_refused(layers):
    step, x = make()
    for bad in (x, x.float()):
        for call in calls(layers, step, bad):
            with pytest.raises(ValueError, match="BF16 hidden states on the GPU"):
                call()
