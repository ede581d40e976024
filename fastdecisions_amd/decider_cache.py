"""Caches of decider requests: score many questions over one prefix, feed prompts in pieces, extend by tokens.

The reference computes a shared prefix once and forks its cache per question (keys and values,
conv state, recurrent state; ref: src/decider/shared_prefix.py:157-200).  ``DeciderCache`` holds
the caches of up to ``requests`` requests of one model:

* attention layers — a pool of pages of keys and values, bf16, e4m3 with a power-of-two scale
  per token and head, or 4-bit with one per 32 features (``paged_kv_kernel``); a request holds pages, not a range, so a fork shares
  its parent's whole pages and copies the last, partly filled one;
* Gated-DeltaNet layers — the conv's last inputs and the fp32 state of the delta rule, a row of a
  pool per request.

Use (``model`` with every HIP kernel installed, inference mode)::

    cache = DeciderCache(model.shape, requests=64, tokens=200_000)
    prefix = cache.open()
    model.hidden(ids, cache=cache.step([prefix], [ids.shape[1]]))       # fill, in one or more pieces
    forks = [cache.fork(prefix) for _ in questions]
    step = cache.step(forks, lengths)                                   # one packed row [1, sum(lengths)]
    logits = model(packed_ids, cache=step)

A step reserves its pages and counts its tokens when it is made; run each step once, in order, or
take it back with ``CacheStep.cancel``: the rows of a step that is never run are whatever its pages
held before.  A forward that refuses its step leaves it waiting, and its requests take no other step
and no fork before it is run or cancelled; one that fails on the way leaves requests whose layers
hold different tokens, which can only be closed.
With ``key_weights=True`` the attention layers also sum the attention weight that each cached key has drawn
(``paged_evict_kernel``; of every step's tokens, or of its ``observe`` last ones per request), and ``evict`` cuts
requests to the keys that drew most and the most recent ones: a prefix of thousands of tokens, cut once, is
forked as before.  A request's next tokens have the positions behind all the tokens that it has seen
(``position``), however few it holds (``length``).  ``evict`` refuses requests with a step that has not run: its
keys' rows are whatever their pages held before.

``CacheStep.again`` makes the next step of the same shape in the same device tensors, so a
captured forward over a step can be replayed token after token.

Streams: a cache's calls change its tensors (``open`` clears states, ``fork`` copies pages and states,
``evict`` moves keys, ``step`` and ``again`` write the step's tensors) and its host records at once: ``close`` and ``evict`` give pages and
states to whoever opens next, also while a forward that reads them is still queued.  So make all calls,
forwards and replays on one stream, or order the streams yourself: the stream of a later call waits
(``Stream.wait_stream``) for the one of every forward and replay before it, over any request, and
``again`` for the one that still reads its step.  Requests in disjoint steps may run on two streams
at once as long as none of the calls above is made between them without that order.  A cache is not for two threads.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from weakref import WeakSet

import torch

from .model import DeciderShape
from .paged_kv_kernel import SCALE_BLOCK


@dataclass(eq=False)
class CacheStep:
    """New tokens of some requests, packed into one row: what the cached layers need of them."""
    cache: "DeciderCache"
    slots: list[int]
    new: list[int]
    cu_seqlens: torch.Tensor      # int32 [n + 1]
    cache_lens: torch.Tensor      # int32 [n], the new tokens included
    state_indices: torch.Tensor   # int32 [n]
    page_table: torch.Tensor      # int32 [n, max_pages]
    positions: torch.Tensor       # int32 [1, total]
    buffer: torch.Tensor = field(repr=False)
    held: list[list[int]] = field(repr=False)  # the requests' pages; another request of a number has another list
    opened: list[int] = field(repr=False)      # which requests of the cache they are, counted as they were opened
    ends: list[int]               # tokens of each request, the new ones included
    live: bool = True             # neither taken back nor failed
    begun: bool = False           # a forward over it has reached the layers
    ran: bool = False             # a forward over it has run
    captured: bool = False        # a forward over it is in a graph: its runs are replays, which are not seen here
    waiting: bool = False         # a forward over it was refused
    written: bool = False         # an attention layer was called with it, by the model or by itself

    @property
    def max_new(self) -> int:
        return max(self.new)

    @property
    def last_rows(self) -> list[int]:
        """Row of every request's last new token in the packed row."""
        rows, at = [], 0
        for n in self.new:
            at += n
            rows.append(at - 1)
        return rows

    def again(self) -> "CacheStep":
        """The next step of the same requests with as many new tokens each, in the same device tensors."""
        self._check()
        sizes = self.cache._reserve(self.slots, self.new)
        try:
            self.buffer.copy_(sizes)
        except BaseException:
            self.cache._release(self.slots, self.new)
            raise
        self.ends = [self.cache._lens[slot] for slot in self.slots]
        self.written &= not self.ran  # (calls of single layers leave no other sign)
        self.live, self.ran = True, False
        return self

    def cancel(self) -> None:
        """Take back a step that has not run and is the last one of its requests, which then are as before it.  Requests
        whose keys were evicted since hold some that are never computed: they can only be closed."""
        if not self.live:
            raise RuntimeError("The step was cancelled already, or has failed")
        if self.ran:
            raise RuntimeError("The step has run: the states of its requests hold its tokens")
        mine = [i for i, slot in enumerate(self.slots) if self.cache._pages.get(slot) is self.held[i]]  # not closed since
        if any(self.cache._lens[self.slots[i]] != self.ends[i] for i in mine):
            raise RuntimeError("Only the last step of its requests can be cancelled")
        first = [(self.ends[i] - self.new[i]) // self.cache.page_size for i in mine]  # page of the step's first token
        if any(self.cache._users[page] > 1 for i, at in zip(mine, first) for page in self.held[i][at:]):
            raise RuntimeError("A fork of one of its requests holds tokens of the step")
        self.cache._release([self.slots[i] for i in mine], [self.new[i] for i in mine])
        self.cache._lost.update(slot for i, slot in enumerate(self.slots)
                                if i not in mine and self.cache._opened.get(slot) == self.opened[i])
        self.live = False
        self._settle()

    def _check(self) -> None:
        """Refuse a step whose requests are not those it was made for: its pages may be another request's by now."""
        for slot, pages in zip(self.slots, self.held):
            if self.cache._pages.get(slot) is not pages:
                raise ValueError(f"Request {slot} of the step was closed, or keys of it were evicted")

    # ---- what a forward over the step tells it

    def _start(self) -> None:
        self._check()
        if not self.live:
            raise RuntimeError("The step was cancelled or has failed; make another one")
        self.cache._check(self.slots, self)

    def _done(self) -> None:
        if not torch.compiler.is_compiling() and self._capturing():
            self.captured = True
        else:
            self.ran = True
        if self.waiting:
            self._settle()

    def _failed(self) -> None:
        """After an error of a forward.  Before the layers nothing was computed; while a graph is captured nothing runs."""
        if not self.live or any(self.cache._pages.get(slot) is not pages for slot, pages in zip(self.slots, self.held)):
            return
        if self.begun:
            if not self._capturing():
                self.cache._lost.update(self.slots)
                self.live = False
            else:
                self.written = False
        elif not (self.ran or self.captured):
            self.waiting = True
            for slot, end in zip(self.slots, self.ends):
                steps = self.cache._waiting.setdefault(slot, [])
                if self not in steps:  # in the order of their tokens
                    steps.insert(sum(step._end(slot) < end for step in steps), self)

    def _end(self, slot) -> int:
        return self.ends[self.slots.index(slot)]

    def _pending(self) -> bool:
        """No forward has run over it or is in a graph, and one may come.  (None does over a cache in host memory: its steps
        keep the books alone.)"""
        return self.live and not (self.ran or self.captured or self.written) and self.positions.is_cuda

    def __del__(self):
        if self._pending():
            self.cache._dropped.update(zip(self.slots, self.opened))

    def _capturing(self) -> bool:
        return self.positions.is_cuda and torch.cuda.is_current_stream_capturing()

    def _settle(self) -> None:
        """No longer waiting."""
        self.waiting = False
        for slot in self.slots:
            steps = self.cache._waiting.get(slot, [])
            if self in steps:
                steps.remove(self)
                if not steps:
                    del self.cache._waiting[slot]


class DeciderCache:
    def __init__(self, shape: DeciderShape, *, requests: int, tokens: int, max_tokens: int | None = None,
                 page_size: int = 64, kv_dtype: torch.dtype = torch.bfloat16, key_weights: bool = False,
                 observe: int | None = None, device="cuda"):
        """``tokens``: cached tokens of all requests together (rounded up to pages, plus one partly filled
        page per request); ``max_tokens``: of one request (default ``tokens``), the width of the page tables.  A
        step writes its requests' tables whole: 64 of 3125 pages cost it 5.2 ms of host time, of 128 pages 0.33 ms.
        ``key_weights``: sum the attention weight of every cached key, for ``evict``.  The sums take 4 bytes per attention
        layer, request, key head and token of ``max_tokens``, whatever the requests hold: 64 requests of up to 200,000
        tokens (7 layers, 4 heads) 1.4 GB, twice their 4-bit pages; of up to 8192 59 MB.  Give ``max_tokens``: tokens one by
        one are weighed fastest while query heads * requests of a step * ``max_tokens`` stay within 2^26 (64 requests of 256
        to 8192 keys in 4 bits: 22 us a layer, beyond that 98).  ``observe``: of the last ``observe`` tokens of a step's
        requests (default: all)."""
        if requests < 1 or tokens < 1:
            raise ValueError("requests and tokens must be positive")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be a power of two in [16, 256]")
        if kv_dtype not in (torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2):
            raise ValueError("kv_dtype must be bfloat16, float8_e4m3fn or float4_e2m1fn_x2")
        if observe is not None and (observe < 1 or not key_weights):
            raise ValueError("observe must be positive and needs key_weights")
        max_tokens = tokens if max_tokens is None else max_tokens
        self.shape, self.page_size, self.kv_dtype, self.device = shape, page_size, kv_dtype, torch.device(device)
        self.requests = requests
        self.max_pages = -(-max_tokens // page_size)
        self.n_pages = -(-tokens // page_size) + requests
        layers = range(shape.num_hidden_layers)
        attention = [i for i in layers if (i + 1) % shape.full_attention_interval == 0]
        linear = [i for i in layers if (i + 1) % shape.full_attention_interval]
        self._attention = {layer: i for i, layer in enumerate(attention)}
        self._linear = {layer: i for i, layer in enumerate(linear)}
        kv = (len(attention), self.n_pages, shape.num_key_value_heads, page_size, shape.head_dim)
        codes4 = kv_dtype == torch.float4_e2m1fn_x2  # two features a byte, a scale per 32 of them
        pool = lambda: (torch.zeros((*kv[:4], kv[4] // 2), dtype=torch.uint8, device=self.device).view(kv_dtype) if codes4
                        else torch.zeros(kv, dtype=kv_dtype, device=self.device))
        self.k, self.v = pool(), pool()
        self.device = self.k.device                   # with its index: steps go there whatever device is current
        self.k_scale = self.v_scale = None
        if kv_dtype != torch.bfloat16:
            scales = (*kv[:4], kv[4] // SCALE_BLOCK) if codes4 else kv[:4]
            self.k_scale = torch.full(scales, 127, dtype=torch.uint8, device=self.device)
            self.v_scale = self.k_scale.clone()
        self.observe = observe
        self.weights = None
        if key_weights:
            self.weights = torch.zeros((len(attention), requests, shape.num_key_value_heads, self.max_pages * page_size),
                                       dtype=torch.float32, device=self.device)
        heads, dim = shape.linear_num_heads, shape.linear_head_dim
        self.conv = torch.zeros((len(linear), requests, shape.conv_kernel - 1, 3 * heads * dim), dtype=torch.bfloat16,
                                device=self.device)
        self.delta = torch.zeros((len(linear), requests, heads, dim, dim), dtype=torch.float32, device=self.device)
        self._free_slots = list(range(requests))[::-1]
        self._free_pages = list(range(self.n_pages))[::-1]
        self._users = [0] * self.n_pages              # requests that hold a page
        self._pages: dict[int, list[int]] = {}        # of an open request
        self._lens: dict[int, int] = {}               # keys it holds
        self._seen: dict[int, int] = {}               # tokens it has seen: the position of its next one
        self._opened: dict[int, int] = {}             # open requests, counted as they were opened
        self._steps: WeakSet[CacheStep] = WeakSet()   # those that somebody holds
        self._dropped: dict[int, int] = {}            # requests (as in _opened) whose step was dropped before it had run
        self._opens = 0
        self._waiting: dict[int, list[CacheStep]] = {}  # the refused steps of an open request, in order
        self._lost: set[int] = set()                  # open requests that a failed forward left half computed

    # ---- requests

    def open(self) -> int:
        """A new, empty request; its number."""
        if not self._free_slots:
            raise RuntimeError(f"All {self.requests} requests of the cache are open")
        slot = self._free_slots.pop()
        self.conv[:, slot].zero_()
        self.delta[:, slot].zero_()
        if self.weights is not None:
            self.weights[:, slot].zero_()
        self._enter(slot, [], 0, 0)
        return slot

    def fork(self, parent: int) -> int:
        """A new request that continues where ``parent`` stands: whole pages shared, the rest copied."""
        self._check([parent])
        n, pages = self._lens[parent], self._pages[parent]
        whole = n // self.page_size
        if not self._free_slots:
            raise RuntimeError(f"All {self.requests} requests of the cache are open")
        if whole < len(pages) and not self._free_pages:
            raise RuntimeError("The cache has no free page")
        slot = self._free_slots.pop()
        own = pages[:whole]
        for page in own:
            self._users[page] += 1
        if whole < len(pages):
            page = self._take()
            for t in (self.k, self.v, self.k_scale, self.v_scale):
                if t is not None:
                    t.view(torch.uint8)[:, page] = t.view(torch.uint8)[:, pages[whole]]
            own = own + [page]
        self.conv[:, slot] = self.conv[:, parent]
        self.delta[:, slot] = self.delta[:, parent]
        if self.weights is not None:
            self.weights[:, slot] = self.weights[:, parent]
        self._enter(slot, list(own), n, self._seen[parent])
        return slot

    def _enter(self, slot, pages, length, seen) -> None:
        self._pages[slot], self._lens[slot], self._seen[slot], self._opened[slot] = pages, length, seen, self._opens
        self._opens += 1

    def close(self, slot: int) -> None:
        """End a request; pages nobody else holds become free."""
        self._check_open([slot])
        self._give(self._pages.pop(slot))
        del self._lens[slot], self._seen[slot], self._opened[slot]
        self._lost.discard(slot)
        self._waiting.pop(slot, None)
        self._free_slots.append(slot)

    def length(self, slot: int) -> int:
        """Keys that a request holds."""
        self._check_open([slot])
        return self._lens[slot]

    def position(self, slot: int) -> int:
        """Tokens that a request has seen: the position of its next one."""
        self._check_open([slot])
        return self._seen[slot]

    def evict(self, slots: list[int], keep: int, *, recent: int = 0) -> None:
        """Cut requests to ``keep`` keys: in every attention layer and key head the ``recent`` last ones and of the others
        those that drew most attention.  A request that holds no more stays as it is.  The kept keys move to free pages
        (``keep`` tokens of each request, before the old ones become free; requests may be cut one by one); pages that
        forks share stay theirs.  Steps made before are refused afterwards, and so must be the replays of captured ones; a
        step that has not run is run or cancelled first."""
        from .cached_ops import paged_kv_evict_op
        slots, keep, recent = list(slots), int(keep), int(recent)
        if self.weights is None:
            raise RuntimeError("The cache has no key weights: make it with key_weights=True")
        if keep < 1 or not 0 <= recent <= keep:
            raise ValueError("keep must be positive and recent in [0, keep]")
        self._check(slots)
        if len(set(slots)) != len(slots):
            raise ValueError("A request appears once in an eviction")
        cut = [slot for slot in slots if self._lens[slot] > keep]
        if not cut:
            return
        for slot in cut:
            if self._dropped.get(slot) == self._opened[slot]:
                raise RuntimeError(f"A step of request {slot} was dropped before it had run: its keys cannot be chosen from")
        for step in self._steps:
            for slot, pages in zip(step.slots, step.held):
                if slot in cut and self._pages[slot] is pages and step._pending():
                    raise RuntimeError(f"A step of request {slot} has not run: run it or cancel it before its keys are evicted")
        if len(cut) * self.shape.num_key_value_heads * keep >= 1 << 27:  # (refused by the first layer, it would cost the requests)
            raise ValueError("requests * Hkv * keep must be below 2^27: cut fewer requests at once")
        need = -(-keep // self.page_size)
        if need * len(cut) > len(self._free_pages):
            raise RuntimeError(f"The cache has {len(self._free_pages)} free pages, the eviction needs {need * len(cut)}")
        n = len(cut)
        old = max(len(self._pages[slot]) for slot in cut)
        tables = [self._pages[slot] + [-1] * (old - len(self._pages[slot])) for slot in cut]
        new = [[self._take() for _ in range(need)] for _ in cut]
        begun = False
        try:
            sizes = torch.tensor([*sum(tables, []), *sum(new, []), *(self._lens[slot] for slot in cut), *cut], dtype=torch.int32)
            table, new_table, lens, rows = sizes.to(self.device).split([n * old, n * need, n, n])
            for layer in self._attention:
                k, v, k_scale, v_scale = self.attention_layer(layer)
                begun = True
                paged_kv_evict_op(k, v, table.view(n, old), lens, self.key_weights(layer), new_table.view(n, need), keep, recent,
                                  k_scale, v_scale, rows)
        except BaseException:
            for pages in new:
                self._give(pages)
            if begun:  # some layers' weights have moved, others' have not
                self._lost.update(cut)
            raise
        for slot, pages in zip(cut, new):
            self._give(self._pages[slot])
            self._pages[slot], self._lens[slot] = pages, keep

    # ---- steps

    def step(self, slots: list[int], new: list[int]) -> CacheStep:
        """``new[i]`` (>= 1) further tokens of request ``slots[i]``, packed in this order into one row."""
        slots, new = list(slots), [int(n) for n in new]
        if len(slots) != len(new) or not slots or min(new) < 1:
            raise ValueError("A step takes one or more requests and a positive number of new tokens of each")
        sizes = self._reserve(slots, new)
        try:
            buffer = sizes.to(self.device)
        except BaseException:  # out of memory
            self._release(slots, new)
            raise
        n, total = len(slots), sum(new)
        cu, lens, idx, table, pos = buffer.split([n + 1, n, n, n * self.max_pages, total])
        step = CacheStep(self, slots, new, cu, lens, idx, table.view(n, self.max_pages), pos.view(1, total), buffer,
                         [self._pages[slot] for slot in slots], [self._opened[slot] for slot in slots],
                         [self._lens[slot] for slot in slots])
        self._steps.add(step)
        return step

    def _check_open(self, slots) -> None:
        for slot in slots:
            if slot not in self._lens:
                raise ValueError(f"{slot} is no open request of the cache")

    def _check(self, slots, step=None) -> None:
        """Refuse requests that are not open, or that hold tokens (before those of ``step``) no forward has computed."""
        self._check_open(slots)
        for slot in slots:
            if slot in self._lost:
                raise RuntimeError(f"A forward over request {slot} failed on the way; it can only be closed")
            if slot in self._waiting and (step is None or self._waiting[slot][0]._end(slot) < step._end(slot)):
                raise RuntimeError(f"A step of request {slot} was refused and has not run: run it or cancel it")

    def _take(self) -> int:
        page = self._free_pages.pop()
        self._users[page] = 1
        return page

    def _give(self, pages) -> None:
        for page in pages:
            self._users[page] -= 1
            if self._users[page] == 0:
                self._free_pages.append(page)

    def _release(self, slots, new) -> None:
        """Undo ``_reserve`` of the requests' last tokens."""
        for slot, n in zip(slots, new):
            self._lens[slot] -= n
            self._seen[slot] -= n
            pages = -(-self._lens[slot] // self.page_size)
            self._give(self._pages[slot][pages:][::-1])
            del self._pages[slot][pages:]

    def _reserve(self, slots, new) -> torch.Tensor:
        """Pages for the new tokens; the step's device tensors as one host tensor."""
        self._check(slots)
        if len(set(slots)) != len(slots):
            raise ValueError("A request appears once in a step")
        need = []
        for slot, n in zip(slots, new):
            pages = -(-(self._lens[slot] + n) // self.page_size)
            if pages > self.max_pages:
                raise RuntimeError(f"Request {slot} would pass the cache's {self.max_pages * self.page_size} tokens per request")
            need.append(pages - len(self._pages[slot]))
        if sum(need) > len(self._free_pages):
            raise RuntimeError(f"The cache has {len(self._free_pages)} free pages, the step needs {sum(need)}")
        cu, lens, table, pos = [0], [], [], []
        for slot, n, pages in zip(slots, new, need):
            held, seen = self._lens[slot], self._seen[slot]
            self._pages[slot] += [self._take() for _ in range(pages)]
            self._lens[slot], self._seen[slot] = held + n, seen + n
            cu.append(cu[-1] + n)
            lens.append(held + n)
            table += self._pages[slot] + [-1] * (self.max_pages - len(self._pages[slot]))
            pos += range(seen, seen + n)
        return torch.tensor(cu + lens + list(slots) + table + pos, dtype=torch.int32)

    # ---- what the layers see

    def attention_layer(self, layer: int):
        """(k, v, k_scale, v_scale) of an attention layer's cache."""
        i = self._attention[layer]
        scales = (None, None) if self.k_scale is None else (self.k_scale[i], self.v_scale[i])
        return self.k[i], self.v[i], *scales

    def key_weights(self, layer: int):
        """Attention weight that an attention layer's cached keys have drawn, [requests, Hkv, max_tokens] (None without
        ``key_weights``)."""
        return None if self.weights is None else self.weights[self._attention[layer]]

    def linear_layer(self, layer: int):
        """(conv state pool, delta state pool) of a Gated-DeltaNet layer."""
        i = self._linear[layer]
        return self.conv[i], self.delta[i]

    def read(self, slot: int, layer: int):
        """Keys and values [1, Hkv, length, D] (bf16) that an attention layer has cached of a request."""
        from .cached_ops import paged_kv_read_op
        self._check([slot])
        n, pages = self._lens[slot], self._pages[slot]
        k, v, k_scale, v_scale = self.attention_layer(layer)
        table = torch.tensor([pages or [-1]], dtype=torch.int32).to(self.device)
        cu = torch.tensor([0, n], dtype=torch.int32).to(self.device)
        return paged_kv_read_op(k, v, table, cu, n, k_scale, v_scale)


def cached_layers_ready(core) -> bool:
    """True when every layer's cached forward can run: attention and Gated-DeltaNet patched, the delta
    rule's heads 128 wide."""
    for layer in core.layers:
        attention, linear = getattr(layer, "self_attn", None), getattr(layer, "linear_attn", None)
        if attention is not None and not (hasattr(attention, "_native_gqa_original_forward")
                                          and attention.head_dim in (64, 128, 256)):
            return False
        if linear is not None and not (
                hasattr(linear, "_packed_original_forward") and getattr(linear, "_fd_gated_delta", False)
                and linear.key_dim == linear.value_dim and linear.head_k_dim == linear.head_v_dim == 128
                and linear.conv1d.bias is None and linear.activation == "silu" and 2 <= linear.conv_kernel_size <= 4):
            return False
    return True


def check_cached_call(layer, hidden_states, **others) -> None:
    """Refuse what a layer's forward over a ``CacheStep`` does not compute: gradients, dropout, other devices and
    types, and masks or caches (``others``) beside the step."""
    if torch.is_grad_enabled():
        raise RuntimeError("The cached forward is for inference: call it without gradients (torch.no_grad() or "
                           "torch.inference_mode())")
    if layer.training and getattr(layer, "attention_dropout", 0.0):
        raise RuntimeError("The cached forward has no dropout: call it in eval mode")
    if not hidden_states.is_cuda or hidden_states.dtype != torch.bfloat16:
        raise ValueError("The cached forward takes BF16 hidden states on the GPU")
    for name, value in others.items():
        if value is not None:
            raise ValueError(f"{name} has no meaning beside fd_cache: a step's tokens see everything their requests hold")
