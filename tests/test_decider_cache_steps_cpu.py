"""Steps of a DeciderCache that are not run as they were made: their requests closed, their forwards refused or
failed (no GPU)."""
from __future__ import annotations

import pytest
import torch

from fastdecisions_amd.decider_cache import DeciderCache
from fastdecisions_amd.model import TINY, build_decider


@pytest.fixture(scope="module")
def model():
    return build_decider(TINY, seed=1, device="cpu")


def make(**kw):
    return DeciderCache(TINY, **(dict(requests=3, tokens=200, max_tokens=100, page_size=16, device="cpu") | kw))


def ids(n):
    return torch.zeros((1, n), dtype=torch.long)


@torch.no_grad()
def test_a_step_of_a_closed_request(model):
    """Its number and its pages may be another request's."""
    c = make()
    a, b = c.open(), c.open()
    step = c.step([a, b], [20, 3])
    c.close(a)
    other = c.open()
    assert other == a
    taken = c.step([other], [5])
    for use in (step.again, lambda: model(ids(23), cache=step)):
        with pytest.raises(ValueError, match="was closed"):
            use()
    assert c.length(other) == 5 and c.length(b) == 3
    assert taken.again() is taken and c.length(other) == 10
