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


def state_of(c):
    return (dict(c._lens), {s: list(p) for s, p in c._pages.items()}, sorted(c._free_pages), list(c._users))


@torch.no_grad()
def test_a_refused_forward_leaves_its_step_waiting(model):
    """Its tokens were counted and never computed: whatever continues the request would attend over what its new
    pages held before."""
    c = make()
    a, b = c.open(), c.open()
    c.step([a], [20])
    before = state_of(c)
    step = c.step([a, b], [30, 5])
    with pytest.raises(ValueError, match="ids"):
        model(ids(34), cache=step)
    for use in (lambda: c.step([a], [1]), lambda: c.step([b], [1]), lambda: c.fork(a), step.again, lambda: c.read(b, 3)):
        with pytest.raises(RuntimeError, match="run it or cancel it"):
            use()
    with pytest.raises(RuntimeError, match="install_hip_kernels"):  # it may be tried again
        model(ids(35), cache=step)
    step.cancel()
    assert state_of(c) == before and not c._waiting
    with pytest.raises(RuntimeError, match="make another"):
        model(ids(35), cache=step)
    assert c.length(a) == 20 and c.length(b) == 0
    c.step([a], [1])
    c.fork(b)
    assert step.again() is step and c.length(a) == 51 and step.positions[0, :30].tolist() == list(range(21, 51))


@torch.no_grad()
def test_an_earlier_refused_step_holds_back_the_later_one(model):
    c = make()
    a = c.open()
    first, second = c.step([a], [3]), c.step([a], [2])
    with pytest.raises(ValueError):
        model(ids(9), cache=first)
    with pytest.raises(RuntimeError, match="run it or cancel it"):
        model(ids(2), cache=second)
    with pytest.raises(RuntimeError, match="Only the last"):
        first.cancel()
    second.cancel()
    first.cancel()
    assert c.length(a) == 0 and len(c._free_pages) == c.n_pages


@torch.no_grad()
def test_a_forward_that_fails_on_the_way(model):
    """Some layers hold the step's tokens, others do not: nothing may continue the request."""
    c = make()
    a, b = c.open(), c.open()
    step, other = c.step([a], [3]), c.step([b], [4])
    step.begun = True
    step._failed()                                         # an error behind the first layer
    for use in (lambda: c.step([a], [1]), lambda: c.fork(a), step.again, lambda: c.read(a, 3)):
        with pytest.raises(RuntimeError, match="only be closed"):
            use()
    with pytest.raises(RuntimeError, match="failed"):
        step.cancel()
    c.close(a)
    a = c.open()
    c.step([a], [1])
    other.cancel()
    assert c.length(b) == 0


@torch.no_grad()
def test_what_has_run_stays(model):
    """A refused repetition of a step takes nothing back."""
    c = make()
    a = c.open()
    step = c.step([a], [3])
    step._done()                                           # as after a forward
    with pytest.raises(ValueError):
        model(ids(4), cache=step)
    with pytest.raises(RuntimeError, match="has run"):
        step.cancel()
    assert c.length(a) == 3
    step.again()
    step.cancel()
    assert c.length(a) == 3
    both = c.step([a, c.open()], [2, 2])
    with pytest.raises(ValueError):
        model(ids(1), cache=both)
    c.close(a)                                             # the other request is still held by the step
    both.cancel()
    assert len(c._free_pages) == c.n_pages and not c._waiting


@pytest.mark.parametrize("where", ["to", "copy_"])
def test_a_step_that_finds_no_memory(where, monkeypatch):
    """The tokens of a step that was never handed out would be counted for good."""
    c = make()
    a = c.open()
    step = c.step([a], [20])
    before = state_of(c)

    def full(*args, **kwargs):
        raise RuntimeError("out of memory")
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, where, full)
        with pytest.raises(RuntimeError, match="out of memory"):
            c.step([a], [40]) if where == "to" else step.again()
    assert state_of(c) == before
    assert step.again().positions.tolist() == [list(range(20, 40))]


def test_a_forked_step_is_not_taken_back():
    """The request would write its next tokens into a page that the fork reads."""
    c = make()
    a = c.open()
    c.step([a], [20])
    step = c.step([a], [30])
    b = c.fork(a)
    with pytest.raises(RuntimeError, match="fork"):
        step.cancel()
    c.close(b)
    step.cancel()
    assert c.length(a) == 20 and len(c._pages[a]) == 2
    b = c.fork(a)                                          # one whole page shared, 20 tokens in both
    step = c.step([a], [30])
    step.cancel()
    assert c.length(a) == c.length(b) == 20 and c._pages[a][0] == c._pages[b][0]


@torch.no_grad()
def test_refused_steps_wait_in_order(model):
    """The second of two refused steps still waits when the first has run."""
    c = make()
    a, b = c.open(), c.open()
    first, second = c.step([a], [3]), c.step([a, b], [2, 1])
    for step in (second, first, second):
        with pytest.raises(ValueError, match="ids"):
            model(ids(9), cache=step)
    with pytest.raises(RuntimeError, match="run it or cancel it"):
        model(ids(3), cache=second)
    first._done()                                          # as after a forward
    with pytest.raises(RuntimeError, match="run it or cancel it"):
        c.step([a], [1])
    with pytest.raises(RuntimeError, match="install_hip_kernels"):  # it is its turn
        model(ids(3), cache=second)
    second.cancel()
    assert c.length(a) == 3 and c.length(b) == 0 and not c._waiting
    first, second = c.step([a], [1]), c.step([a], [2])
    with pytest.raises(ValueError, match="ids"):
        model(ids(9), cache=second)
    with pytest.raises(RuntimeError, match="install_hip_kernels"):  # a refused later step holds nothing back before it
        model(ids(1), cache=first)
