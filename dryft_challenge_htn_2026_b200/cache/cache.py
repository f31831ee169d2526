"""The cache of a model: a slot per live sequence, and per group of layers either paged keys and
values or a fixed-size state.

Layers (cache entries) whose mixers make the same request share a group; each group has storage
and, for keys/values, a page pool of its own, so a group of windowed layers can give pages back
that a group of full-attention layers must keep. A sequence's length is the same in every group.

Key/value storage of a group: [entries, 2 (k, v), pages, n_kv_heads, PAGE, head_dim]; page p of a
kv head is one contiguous [PAGE, head_dim] tile. State storage: [entries, slots, *shape].
The reference keeps one dense [B, nkv, cap, hd] pair per layer per batch shape
(engine/engine.py:344-347); pages let sequences of any lengths share one allocation.
"""
from dataclasses import dataclass

import numpy as np
import torch

from ..csrc import api
from ..csrc.api import PAGE
from .pool import CacheFull, PagePool, SlotTable
from .requests import KVRequest, StateRequest


@dataclass
class KVView:
    group: int            # index into StepContext.tables
    k: torch.Tensor       # [pages, n_kv, PAGE, hd]
    v: torch.Tensor


@dataclass
class StateView:
    group: int
    state: torch.Tensor   # [slots, *shape]; row = the sequence's slot (StepContext.seq_slot)


class KVGroup:
    def __init__(self, index, request, entries, num_pages, device, allocate=True):
        self.index, self.request, self.entries = index, request, list(entries)
        self.pool = PagePool(num_pages)
        self.pages = {}                                   # slot -> list of page ids (-1: given back)
        self.first = {}                                   # slot -> index of the first page not yet given back
        self.store = self.v_store = None
        vd = request.v_head_dim
        self.keys_only = bool(request.values_in_keys)
        if self.keys_only:
            if vd is None or vd > request.head_dim:
                raise ValueError(f"values of {vd} numbers inside key rows of {request.head_dim}")
            if allocate:
                self.store = torch.zeros((len(self.entries), num_pages, request.n_kv_heads, PAGE, request.head_dim),
                                         dtype=request.dtype, device=device)
        elif allocate and (vd is None or vd == request.head_dim):
            self.store = torch.zeros((len(self.entries), 2, num_pages, request.n_kv_heads, PAGE, request.head_dim),
                                     dtype=request.dtype, device=device)
        elif allocate:    # keys and values of different sizes: a store each, [entries, pages, n_kv, PAGE, size]
            self.store = torch.zeros((len(self.entries), num_pages, request.n_kv_heads, PAGE, request.head_dim),
                                     dtype=request.dtype, device=device)
            self.v_store = torch.zeros((len(self.entries), num_pages, request.n_kv_heads, PAGE, vd),
                                       dtype=request.dtype, device=device)

    def view(self, entry):
        e = self.entries.index(entry)
        if self.keys_only:
            return KVView(self.index, self.store[e], None)
        if self.v_store is not None:
            return KVView(self.index, self.store[e], self.v_store[e])
        return KVView(self.index, self.store[e, 0], self.store[e, 1])

    def start(self, slot):
        self.pages[slot] = []
        self.first[slot] = 0

    def ensure(self, slot, length):
        """Pages for positions [0, length) of the slot (those still inside the window)."""
        have = self.pages[slot]
        need = (length + PAGE - 1) // PAGE - len(have)
        if need > 0:
            have.extend(self.pool.alloc(need))

    def trim(self, slot, length):
        """Gives back pages no later token can see: a query at position >= length reads keys
        > length - window - 1 only, and with a chunk mask none before the chunk that holds position
        ``length`` (later queries sit in that chunk or a later one)."""
        w, c = self.request.window, self.request.chunk
        if w is None and c is None:
            return
        first_needed = 0 if w is None else length - w + 1
        if c is not None:
            first_needed = max(first_needed, length // c * c)
        have = self.pages[slot]
        i = max(self.first[slot], (self.request.keep_first + PAGE - 1) // PAGE)   # the kept first positions' pages stay
        while i < len(have) and i * PAGE + PAGE - 1 < first_needed:
            self.pool.free([have[i]])
            have[i] = -1
            i += 1
        self.first[slot] = i

    def end(self, slot):
        self.pool.free([p for p in self.pages.pop(slot) if p >= 0])
        del self.first[slot]

    def stores(self):
        """The tensors [.., pages, n_kv, PAGE, size] that hold the group's rows."""
        return [t for t in (self.store, self.v_store) if t is not None]

    def bytes(self):
        return sum(t.numel() * t.element_size() for t in self.stores())


class StateGroup:
    def __init__(self, index, request, entries, max_slots, device, allocate=True):
        self.index, self.request, self.entries = index, request, list(entries)
        self.store = None
        if allocate:
            self.store = torch.zeros((len(self.entries), max_slots, *request.shape), dtype=request.dtype, device=device)

    def view(self, entry):
        return StateView(self.index, self.store[self.entries.index(entry)])

    def start(self, slot):
        if self.store is not None:
            self.store[:, slot].zero_()

    def ensure(self, slot, length):
        pass

    def trim(self, slot, length):
        pass

    def end(self, slot):
        pass

    def bytes(self):
        return 0 if self.store is None else self.store.numel() * self.store.element_size()


class Cache:
    """``entry_requests``: for each cache entry (in order) the list of requests of its mixer."""

    def __init__(self, entry_requests, max_tokens, max_slots, device, allocate=True):
        self.num_pages = max(1, (max_tokens + PAGE - 1) // PAGE)
        self.max_slots = max(1, min(max_slots, self.num_pages))
        self.slots = SlotTable(self.max_slots)
        self.length = {}                                   # slot -> tokens cached
        self.groups = []
        self._views = []                                   # per entry: list of views, in request order
        by_request = {}
        for entry, requests in enumerate(entry_requests):
            for r in requests:
                by_request.setdefault(r, []).append(entry)
        for r, entries in by_request.items():
            if isinstance(r, KVRequest):
                g = KVGroup(len(self.groups), r, entries, self.num_pages, device, allocate)
            elif isinstance(r, StateRequest):
                g = StateGroup(len(self.groups), r, entries, self.max_slots, device, allocate)
            else:
                raise TypeError(f"unknown cache request {r!r}")
            self.groups.append(g)
        if allocate:
            index = {g.request: g for g in self.groups}
            self._views = [[index[r].view(entry) for r in requests] for entry, requests in enumerate(entry_requests)]

    def views(self, entry):
        return self._views[entry]

    # -- life of a sequence ------------------------------------------------------------------
    def begin(self):
        slot = self.slots.acquire()
        self.length[slot] = 0
        for g in self.groups:
            g.start(slot)
        return slot

    def reserve(self, slot, n_new):
        """Room for n_new more tokens of the slot in every group (before the step that writes them)."""
        try:
            for g in self.groups:
                g.ensure(slot, self.length[slot] + n_new)
        except CacheFull:
            raise CacheFull(f"cache full: sequence in slot {slot} cannot grow from {self.length[slot]} by {n_new} "
                            f"tokens ({self.num_pages} pages of {PAGE} tokens in all)") from None

    def commit(self, slot, n_new):
        """After the step: the tokens are in; windowed groups give back what fell out of sight."""
        self.length[slot] += n_new
        for g in self.groups:
            g.trim(slot, self.length[slot])

    def end(self, slot):
        if slot not in self.length:
            raise ValueError(f"slot {slot} ended but not live")
        for g in self.groups:
            g.end(slot)
        del self.length[slot]
        self.slots.release(slot)

    def page_rows(self, group, slots, min_width=1):
        """Page lists of the slots in one group, padded with -1 to a common width."""
        g = self.groups[group]
        if not isinstance(g, KVGroup):
            return [[-1] * min_width for _ in slots]
        rows = [g.pages[s] for s in slots]
        width = max([min_width] + [len(r) for r in rows])
        return [r + [-1] * (width - len(r)) for r in rows]

    def reorder(self, slots, parents, first=None):
        """Sequences take the places of others, as the beams of a search do: ``slots[r][b]`` is beam b of request r, and gets the rows
        from ``first[r]`` on (None: all) and the states of beam ``parents[r][b]`` as they are now. The beams of a request have equal
        lengths, and rows before ``first[r]`` in common. Moves within the cache, on the current stream."""
        beams = len(slots[0])
        flat = [s for row in slots for s in row]
        if len(set(flat)) != len(flat) or any(len(row) != beams or len(p) != beams for row, p in zip(slots, parents)) or len(slots) != len(parents):
            raise ValueError("a slot of its own for every beam, and as many beams and parents for every request")
        if any(not 0 <= q < beams for p in parents for q in p):
            raise ValueError(f"parents are numbers of the request's {beams} beams")
        length = [self.length[row[0]] for row in slots]
        if any(self.length[s] != n for row, n in zip(slots, length) for s in row):
            raise ValueError("the beams of a request must have equal lengths")
        if all(list(p) == list(range(beams)) for p in parents):
            return
        arrays = [np.array(a, np.int32) for a in (flat, parents, first or [0] * len(slots), length)]
        arrays += [np.array(self.page_rows(g, flat), np.int32) for g in range(len(self.groups)) if isinstance(self.groups[g], KVGroup)]
        store = next(g.store for g in self.groups if g.store is not None)
        dev = torch.from_numpy(np.concatenate([a.reshape(-1) for a in arrays])).to(store.device)
        dev = [t.view(a.shape) for t, a in zip(dev.split([a.size for a in arrays]), arrays)]
        tables = iter(dev[4:])
        for g in self.groups:
            if isinstance(g, KVGroup):
                table = next(tables)
                for t in g.stores():
                    api.kv_reorder(t, table, dev[1], dev[2], dev[3])
            else:
                api.state_reorder(g.store, dev[0], dev[1])

    def state_snapshot(self, slots):
        """Copies of the per-sequence states of ``slots`` (every state group), for a caller that runs a
        step more than once (the warm-up runs before a graph capture) and must leave the states as one run
        would: ``state_restore`` puts them back. Keys and values need none: a repeated step rewrites the
        same cache rows with the same numbers."""
        index = torch.tensor(list(slots), dtype=torch.long, device=self.groups[0].store.device) if self.groups else None
        return [(g, index, g.store[:, index].clone()) for g in self.groups if isinstance(g, StateGroup) and g.store is not None]

    @staticmethod
    def state_restore(snapshot):
        for g, index, saved in snapshot:
            g.store[:, index] = saved

    def pages_held(self, slot):
        """Per key/value group the length of the slot's page list (pages given back included): it
        changes exactly when a step's page tables have to be written anew."""
        return tuple(len(g.pages[slot]) for g in self.groups if isinstance(g, KVGroup))

    def bytes(self):
        return sum(g.bytes() for g in self.groups)

    def pages_free(self):
        return [g.pool.n_free for g in self.groups if isinstance(g, KVGroup)]
