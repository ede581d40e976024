"""Evictions of requests with a step that has not run (no GPU: the kernels' op is replaced)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest

from test_decider_cache_evict_cpu import calls, make  # noqa: F401  (calls: the fixture)
from test_decider_cache_steps_cpu import state_of


def unusable(c, slot):
    for use in (lambda: c.step([slot], [1]), lambda: c.fork(slot), lambda: c.evict([slot], 2), lambda: c.read(slot, 3)):
        with pytest.raises(RuntimeError, match="only be closed"):
            use()


def test_a_step_taken_back_after_an_eviction(calls):  # noqa: F811
    """The kept keys are of tokens that nobody will compute: nothing may attend to them.  The step's other request is as
    before it."""
    c = make()
    a, b = c.open(), c.open()
    c.step([b], [7])
    step = c.step([a, b], [50, 20])
    c.evict([a], 10)
    step.cancel()
    assert (c.length(a), c.length(b), c.position(b)) == (10, 7, 7)
    unusable(c, a)
    c.step([b], [1]).cancel()
    c.close(a)
    assert c.open() == a
    c.step([a], [1])
    c.close(a)
    c.close(b)
    assert len(c._free_pages) == c.n_pages


def test_a_number_that_is_another_request_by_then(calls):  # noqa: F811
    c = make()
    a = c.open()
    step = c.step([a], [50])
    c.evict([a], 10)
    c.close(a)
    assert c.open() == a
    step.cancel()
    c.step([a], [5])
    assert c.length(a) == 5


def on_a_gpu(step):
    """As the steps of a cache whose forwards can run."""
    step.positions = SimpleNamespace(is_cuda=True)
    return step


def test_a_step_that_may_run_holds_back_an_eviction(calls):  # noqa: F811
    c = make()
    a, b = c.open(), c.open()
    c.step([a], [20])
    c.step([b], [30])
    before = state_of(c)
    step = on_a_gpu(c.step([a], [50]))
    held = state_of(c)
    with pytest.raises(RuntimeError, match=f"request {a} has not run"):
        c.evict([b, a], 10)
    assert state_of(c) == held and not calls and not c._lost
    c.evict([a], 70)                                       # nothing to cut
    step.cancel()
    assert state_of(c) == before
    c.evict([a, b], 10)
    assert (c.length(a), c.position(a), c.length(b)) == (10, 20, 10) and calls


@pytest.mark.parametrize("sign", ["ran", "captured", "written"])
def test_a_step_that_has_run_holds_back_nothing(calls, sign):  # noqa: F811
    """Run by the model, recorded into a graph whose replays are not seen, or through layers called by themselves."""
    c = make()
    a = c.open()
    step = on_a_gpu(c.step([a], [30]))
    setattr(step, sign, True)
    c.evict([a], 20)
    assert c.length(a) == 20
    step = on_a_gpu(c.step([a], [2]))
    step.buffer, step.ran, step.written = SimpleNamespace(copy_=lambda sizes: None), True, True
    step.again()                                           # the next one has not
    with pytest.raises(RuntimeError, match="has not run"):
        c.evict([a], 20)
    step.ran = True
    c.evict([a], 20)
    assert (c.length(a), c.position(a)) == (20, 34)


def test_a_failed_step_holds_back_nothing_else(calls):  # noqa: F811
    c = make()
    a, b = c.open(), c.open()
    step = on_a_gpu(c.step([a, b], [30, 30]))
    step.live = False
    c._lost.add(a)
    c.evict([b], 20)
    assert c.length(b) == 20


def test_more_kept_keys_than_an_eviction_moves():
    """Refused before anything has moved, where the kernels' entry point refuses it too: the requests stay as they are."""
    from fastdecisions_amd.decider_cache import DeciderCache
    from fastdecisions_amd.model import TINY
    keep = (1 << 26) // TINY.num_key_value_heads
    c = DeciderCache(TINY, requests=2, tokens=4 * keep + 1024, max_tokens=keep + 1, page_size=256, key_weights=True, device="meta")
    slots = [c.open(), c.open()]
    for s in slots:
        c._pages[s], c._lens[s], c._seen[s] = [c._take() for _ in range(keep // 256 + 1)], keep + 1, keep + 1
    free = len(c._free_pages)
    with pytest.raises(ValueError, match=r"below 2\^27"):
        c.evict(slots, keep)
    assert not c._lost and len(c._free_pages) == free and c.length(slots[0]) == keep + 1


def test_a_dropped_step_holds_back_an_eviction(calls):  # noqa: F811
    """Nobody can run it or take it back any more, as after an error between a step and its forward."""
    c = make()
    a, b = c.open(), c.open()
    c.step([a, b], [5, 30])
    step = on_a_gpu(c.step([a], [50]))
    del step
    with pytest.raises(RuntimeError, match="dropped before it had run"):
        c.evict([b, a], 10)
    assert not calls
    c.evict([b], 10)
    c.close(a)
    assert c.open() == a
    c.step([a], [50])
    c.evict([a], 10)                                       # another request
    for end in ("ran", "live"):                            # run or taken back, then dropped
        step = on_a_gpu(c.step([a], [3]))
        setattr(step, end, end == "ran")
        del step
        c.evict([a], 10)
    assert c.length(a) == 10
