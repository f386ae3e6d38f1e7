"""The cache: a slot per live sequence, paged keys and values per storage group, and a
fixed-size per-sequence state area.

Storage groups. Cache entries (one per schedule entry that writes a cache) with the same need
(kind, K/V heads, head size, window) share a group; each group has its own page pool and its
own device storage ``k, v: [entries, pages, kv_heads, PAGE, head_dim]``. A ``full`` group keeps
every key and value of a sequence; a ``window`` group gives pages back once every position in
them is older than the window (positions left of ``length - window`` are never read again; with
``keep_first`` the pages of a sequence's first positions are held as long as the sequence lives).
The reference's analogues are StaticCache (src/transformers/cache_utils.py:1058-1230: storage
allocated once, written in place), HybridCache (:1550-1743: per-layer kinds with their own
shapes) and MambaCache (:1746-1859: fixed-size state per batch row, reset in place).

Sizing. ``max_tokens`` is the most tokens that live sequences hold at one time, each sequence's
count rounded up to a whole page of 64; every group gets ``max_tokens / 64`` pages.

Sequences. ``open()`` gives a slot, ``reserve(slot, n)`` gets the pages for ``n`` more tokens
(or raises CacheFull before anything is launched), ``commit(slot, n)`` advances the length
after the step, ``close(slot)`` gives pages and slot back. Storage is zeroed when it is
allocated and never again: lengths and page lists gate every read. The state area is zeroed for a slot when it is opened.

Pages are copied, shared and moved by ``fork(slot)`` (another sequence with the same past: whole pages are shared, the partly
filled one and the state are copied), ``truncate(slot, length)`` (the last tokens forgotten, their pages given back),
``compact()`` (the pages that are held become the lowest of the pool) and ``resize(max_tokens)`` (other storage for as many
tokens, with the pages that are held). A shared page is full: no sequence writes to a page that another one holds. The copies
run on the device's current stream, like a step (``kernels.copy_pages``); the reference's analogues are ``crop``,
``batch_repeat_interleave`` and ``reorder_cache`` (src/transformers/cache_utils.py:454-505), which copy whole tensors.

``kv_dtype=torch.float8_e4m3fn`` keeps keys and values as 8-bit codes with an exponent for each page and K/V head (``k_exp``,
``v_exp`` beside ``k``, ``v``): half the bytes of bfloat16 in memory and on the way to the attention, for mixers that say so in
their need (``CacheNeed.eight_bit``) and models in bfloat16.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..parts.base import CacheNeed, StateNeed
from .pool import CacheError, CacheFull, IdPool, SequenceRecord

PAGE = 64

# What a kind of cache entry keeps: for a sequence of `length` tokens, the first position that a later
# query can still see (pages that lie wholly before it go back to the pool after every step).
# ``register_cache_kind`` adds a kind without a change here; the mixer that names it reads accordingly.
CACHE_KINDS = {
    "full": lambda need, length: 0,
    # the next query sits at position >= length and sees keys > position - window
    "window": lambda need, length: max(0, length - need.window + 1),
}


def register_cache_kind(kind: str, first_needed) -> None:
    """``first_needed(need: CacheNeed, length: int) -> int``: the first cached position that queries at
    positions >= length may read."""
    CACHE_KINDS[kind] = first_needed


class StorageGroup:
    def __init__(self, need: CacheNeed, entries: List[int], num_pages: int, dtype: torch.dtype, device,
                 kv_dtype: Optional[torch.dtype] = None):
        if need.kind not in CACHE_KINDS:
            raise ValueError(f"unknown cache kind {need.kind!r} (kinds: {', '.join(sorted(CACHE_KINDS))})")
        if need.kind == "window" and need.window <= 0:
            raise ValueError("a window group needs window > 0")
        if kv_dtype is not None and not need.eight_bit:
            raise ValueError(f"a cache in {str(kv_dtype).replace('torch.', '')} was asked for, but a mixer of this model does not take its "
                             f"pages in 8 bits ({need})")
        self.need, self.kv_dtype, self.dtype, self.device = need, kv_dtype, dtype, device
        self.entries = list(entries)
        self.index_of = {e: i for i, e in enumerate(self.entries)}
        self.pool = IdPool(num_pages, "cache page")
        self.k, self.v, self.k_exp, self.v_exp = self._storage(num_pages)

    def _storage(self, num_pages: int):
        need = self.need
        shape = (len(self.entries), num_pages, need.kv_heads, PAGE, need.head_dim)
        # zeroed once: kernels multiply masked positions of a page by zero, which must not meet a NaN
        dtype = self.dtype if self.kv_dtype is None else self.kv_dtype
        k = torch.zeros(shape, dtype=dtype, device=self.device)
        v_dim = need.head_dim if need.v_head_dim is None else need.v_head_dim
        v = torch.zeros(shape[:-1] + (v_dim,), dtype=dtype, device=self.device)   # no storage with v_head_dim = 0
        if self.kv_dtype is None:
            return k, v, None, None
        return k, v, *(torch.zeros(shape[:3], dtype=torch.int8, device=self.device) for _ in range(2))

    def tensors(self) -> List[torch.Tensor]:
        """All that holds pages: [entries, pages, ...] each."""
        return [t for t in (self.k, self.v, self.k_exp, self.v_exp) if t is not None and t.numel()]

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors())

    def copy_pages(self, src: List[int], dst: List[int], out: Optional[List[torch.Tensor]] = None) -> None:
        if not src:
            return
        if self.k.is_cuda:
            from ..kernels import copy_pages
            copy_pages(self.tensors(), src, dst, out=out)
        else:                # the bookkeeping without a GPU
            for a, b in zip(self.tensors(), out or self.tensors()):
                a, b = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (a, b))
                b[:, dst] = a[:, src]

    def renumber(self, num_pages: int) -> Dict[int, int]:
        """The pages that are held as the lowest of a pool of ``num_pages``; {old: new} of those that moved. Other storage where the
        number changes."""
        if num_pages == self.pool.capacity:
            moved = self.pool.renumber(num_pages)
            self.copy_pages(list(moved), list(moved.values()))
            return moved
        held = [i for i in range(self.pool.capacity) if self.pool.holders(i)]
        fresh = self._storage(num_pages) if num_pages >= len(held) else ()     # allocated before anything changes
        moved = self.pool.renumber(num_pages)
        self.copy_pages(held, [moved.get(i, i) for i in held], out=[t for t in fresh if t is not None and t.numel()])
        _read_by_this_stream(self.tensors())
        self.k, self.v, self.k_exp, self.v_exp = fresh
        return moved


def _read_by_this_stream(tensors) -> None:
    """Storage about to be given up may be on its way to other storage on another stream than the one it was allocated on: its memory is
    nobody else's until the copy has read it."""
    for t in tensors:
        if t.is_cuda:
            t.record_stream(torch.cuda.current_stream(t.device))


class Cache:
    def __init__(self, needs: Sequence[Tuple[int, Optional[CacheNeed], Optional[StateNeed]]], max_tokens: int,
                 dtype: torch.dtype, device, max_slots: Optional[int] = None, kv_dtype: Optional[torch.dtype] = None):
        if max_tokens <= 0:
            raise ValueError(f"max_tokens must be positive, got {max_tokens}")
        if kv_dtype == dtype:
            kv_dtype = None
        if kv_dtype is not None and (kv_dtype != torch.float8_e4m3fn or dtype != torch.bfloat16):
            raise ValueError(f"keys and values are held in the model's dtype, or for a bfloat16 model in float8_e4m3fn; got {kv_dtype} "
                             f"for {dtype}")
        self.num_pages = (max_tokens + PAGE - 1) // PAGE
        self.max_tokens = self.num_pages * PAGE
        self.dtype, self.kv_dtype, self.device = dtype, kv_dtype, torch.device(device)      # kv_dtype None: the model's
        by_need: Dict[CacheNeed, List[int]] = {}
        for entry, need, _ in needs:
            if need is not None:
                by_need.setdefault(need, []).append(entry)
        self.groups: List[StorageGroup] = [StorageGroup(n, es, self.num_pages, dtype, self.device, kv_dtype)
                                           for n, es in by_need.items()]
        self.group_of_entry: Dict[int, int] = {e: gi for gi, g in enumerate(self.groups) for e in g.entries}
        # a live sequence holds at least one page of every group, so pages bound the slots
        self._slots_by_pages = max_slots is None
        self.max_slots = int(max_slots) if max_slots is not None else max(1, min(self.num_pages, 4096))
        self.slots = IdPool(self.max_slots, "sequence slot")
        self.records: Dict[int, SequenceRecord] = {}
        self.epoch = 0   # counts opened and closed sequences: what was planned for an earlier epoch is stale
        self.state_entries: Dict[int, int] = {}
        self.state: Optional[torch.Tensor] = None
        widths = [(e, s.numel) for e, _, s in needs if s is not None and s.numel > 0]
        self.state_offsets: Dict[int, Tuple[int, int]] = {}
        off = 0
        for e, n in widths:
            self.state_offsets[e] = (off, n)
            off += n
        self.state_width = off
        # the state area exists for every model; for one without stateful mixers it has width 0
        self.state = torch.zeros((self.max_slots, self.state_width), dtype=torch.float32, device=self.device)

    # ------------------------------------------------------------------ sequences
    def open(self) -> int:
        (slot,) = self.slots.take(1)
        self.epoch += 1
        self.records[slot] = SequenceRecord(len(self.groups))
        if self.state_width:
            self.state[slot].zero_()
        return slot

    def _record(self, slot: int) -> SequenceRecord:
        try:
            return self.records[slot]
        except KeyError:
            raise CacheError(f"slot {slot} is not open") from None

    def length(self, slot: int) -> int:
        return self._record(slot).length

    def reserve(self, slot: int, n_new: int) -> None:
        """Make sure ``slot`` has pages for ``n_new`` more tokens in every group."""
        rec = self._record(slot)
        if n_new < 0:
            raise ValueError("n_new must be >= 0")
        want = (rec.length + n_new + PAGE - 1) // PAGE
        for gi, g in enumerate(self.groups):
            have = len(rec.pages[gi])
            if want > have:
                rec.pages[gi].extend(g.pool.take(want - have))

    def reserve_all(self, plan: Sequence[Tuple[int, int]]) -> None:
        """Reserve for several sequences at once; if the pages do not suffice, nothing is kept."""
        need = [0] * len(self.groups)
        for slot, n_new in plan:
            rec = self._record(slot)
            want = (rec.length + n_new + PAGE - 1) // PAGE
            for gi in range(len(self.groups)):
                need[gi] += max(0, want - len(rec.pages[gi]))
        for gi, g in enumerate(self.groups):
            if need[gi] > g.pool.available:
                raise CacheFull(f"the step needs {need[gi]} more cache pages of {PAGE} tokens but only "
                                f"{g.pool.available} of {g.pool.capacity} are free (cache sized for "
                                f"{self.max_tokens} tokens)")
        for slot, n_new in plan:
            self.reserve(slot, n_new)

    def commit(self, slot: int, n_new: int) -> None:
        """The step has written ``n_new`` tokens of ``slot``: advance its length, and let window
        groups give back pages that no later query can see."""
        rec = self._record(slot)
        rec.length += n_new
        for gi, g in enumerate(self.groups):
            if rec.length > len(rec.pages[gi]) * PAGE:
                raise CacheError(f"slot {slot} was advanced to {rec.length} tokens beyond its reserved pages")
            first_needed = CACHE_KINDS[g.need.kind](g.need, rec.length)
            if first_needed >= PAGE:
                dead = first_needed // PAGE
                kept = (g.need.keep_first + PAGE - 1) // PAGE     # pages of positions that stay readable for good
                gone = [p for p in rec.pages[gi][kept:dead] if p >= 0]
                if gone:
                    g.pool.give_back(gone)
                    for i in range(kept, dead):
                        rec.pages[gi][i] = -1

    def close(self, slot: int) -> None:
        rec = self._record(slot)
        for gi, g in enumerate(self.groups):
            g.pool.give_back([p for p in rec.pages[gi] if p >= 0])
        del self.records[slot]
        self.epoch += 1
        self.slots.give_back([slot])

    def close_all(self) -> None:
        for slot in list(self.records):
            self.close(slot)

    # ------------------------------------------------------------------ pages copied, shared, given back, moved
    def fork(self, slot: int, share: bool = True) -> int:
        """Another sequence with the past of the one in ``slot``; returns its slot. Whole pages are shared (or copied too, with
        ``share=False``); a partly filled page and the per-sequence state are copied. Raises CacheFull before anything changes."""
        rec = self._record(slot)
        full, rest = divmod(rec.length, PAGE)
        plans = []          # per group: pages to copy, as places in the sequence's list
        for gi, g in enumerate(self.groups):
            places = ([] if share else [i for i in range(full) if rec.pages[gi][i] >= 0]) + ([full] if rest else [])
            if len(places) > g.pool.available:
                raise CacheFull(f"a fork needs {len(places)} more cache pages of {PAGE} tokens but only {g.pool.available} of "
                                f"{g.pool.capacity} are free")
            plans.append(places)
        (new,) = self.slots.take(1)
        self.epoch += 1
        copy = self.records[new] = SequenceRecord(len(self.groups))
        copy.length = rec.length
        for gi, (g, places) in enumerate(zip(self.groups, plans)):
            pages = list(rec.pages[gi][:full + (1 if rest else 0)])
            own = g.pool.take(len(places))
            g.copy_pages([pages[i] for i in places], own)
            for i, p in zip(places, own):
                pages[i] = p
            copied = set(places)
            g.pool.share(p for i, p in enumerate(pages) if p >= 0 and i not in copied)
            copy.pages[gi] = pages
        if self.state_width:
            self.state[new].copy_(self.state[slot])
        return new

    def truncate(self, slot: int, length: int) -> None:
        """Forget the tokens of ``slot`` from ``length`` on and give their pages back (and pages reserved ahead). Not for models with
        per-sequence state, which cannot go back, nor to where a window needs pages that have been given back. Raises before
        anything changes."""
        rec = self._record(slot)
        if not (0 <= length <= rec.length):
            raise ValueError(f"slot {slot} holds {rec.length} tokens: it cannot be cut to {length}")
        if length < rec.length and self.state_width:
            raise CacheError("a sequence with per-sequence state cannot forget its last tokens")
        keep, rest = (length + PAGE - 1) // PAGE, length % PAGE
        for gi, g in enumerate(self.groups):
            first = CACHE_KINDS[g.need.kind](g.need, length) // PAGE
            if any(p < 0 for p in rec.pages[gi][first:keep]):
                raise CacheError(f"slot {slot} cannot be cut to {length} tokens: pages that its window would see again have been given back")
            # the page that the next token goes to, where somebody else holds it as well
            if rest and g.pool.holders(rec.pages[gi][keep - 1]) > 1 and not g.pool.available:
                raise CacheFull(f"cutting slot {slot} to {length} tokens needs a page of its own, and none of {g.pool.capacity} is free")
        for gi, g in enumerate(self.groups):
            pages = rec.pages[gi]
            if rest and g.pool.holders(pages[keep - 1]) > 1:
                (own,) = g.pool.take(1)
                g.copy_pages([pages[keep - 1]], [own])
                g.pool.give_back([pages[keep - 1]])
                pages[keep - 1] = own
            g.pool.give_back([p for p in pages[keep:] if p >= 0])
            del pages[keep:]
        rec.length = length
        self.epoch += 1

    def _renumber(self, num_pages: int) -> int:
        self.epoch += 1      # first: a group may run out of memory after another has moved
        count = 0
        for gi, g in enumerate(self.groups):
            moved = g.renumber(num_pages)
            count += len(moved)
            for rec in self.records.values():
                rec.pages[gi] = [moved.get(p, p) for p in rec.pages[gi]]
        return count

    def compact(self) -> int:
        """Make the pages that are held the lowest of every group's pool; returns how many moved."""
        return self._renumber(self.num_pages)

    def resize(self, max_tokens: int) -> None:
        """Room for ``max_tokens`` tokens in place of what there is: other storage, one group after another, with the pages that are held
        as its lowest. Raises CacheFull before anything changes if they do not fit. Steps captured for the old storage are dropped."""
        if max_tokens <= 0:
            raise ValueError(f"max_tokens must be positive, got {max_tokens}")
        num_pages = (max_tokens + PAGE - 1) // PAGE
        most = max((g.pool.in_use for g in self.groups), default=0)
        if num_pages < most:
            raise CacheFull(f"{most} cache pages of {PAGE} tokens are held, more than {max_tokens} tokens have")
        for name in ("_step_graphs", "_prepared_step"):      # they hold pointers into the old storage
            self.__dict__.pop(name, None)
        self._renumber(num_pages)
        self.num_pages, self.max_tokens = num_pages, num_pages * PAGE
        slots = max(1, min(num_pages, 4096))
        if self._slots_by_pages and slots > self.max_slots:
            state = torch.zeros((slots, self.state_width), dtype=torch.float32, device=self.device)
            state[:self.max_slots] = self.state
            _read_by_this_stream([self.state])
            self.state, self.max_slots = state, slots
            self.slots.grow(slots)

    # ------------------------------------------------------------------ views for the step
    def pages(self, slot: int, group: int) -> List[int]:
        return self._record(slot).pages[group]

    def entry_storage(self, entry: int) -> Tuple[torch.Tensor, torch.Tensor, int]:
        """(K pool, V pool, group index) of a cache entry: pools are [pages, kv_heads, PAGE, head_dim]."""
        gi = self.group_of_entry[entry]
        g = self.groups[gi]
        i = g.index_of[entry]
        return g.k[i], g.v[i], gi

    def entry_exponents(self, entry: int) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """The exponents [pages, kv_heads] of a cache entry's keys and values that are held in 8 bits, or None."""
        g = self.groups[self.group_of_entry[entry]]
        if g.k_exp is None:
            return None
        i = g.index_of[entry]
        return g.k_exp[i], g.v_exp[i]

    def entry_state(self, entry: int) -> Optional[torch.Tensor]:
        """[slots, numel] float32 view of a cache entry's per-sequence state, or None."""
        if entry not in self.state_offsets:
            return None
        off, n = self.state_offsets[entry]
        return self.state[:, off:off + n]

    # ------------------------------------------------------------------ accounting
    def live_tokens(self) -> int:
        return sum(r.length for r in self.records.values())

    def bytes(self) -> int:
        return sum(g.bytes() for g in self.groups) + self.state.numel() * 4

    def check(self) -> None:
        """Invariants: every page of every group is free or held by as many open sequences as the pool says, and one that several
        hold is full in each of them and at the same place."""
        self.slots.check()
        for gi, g in enumerate(self.groups):
            g.pool.check()
            held: Dict[int, List[Tuple[int, bool]]] = {}
            for r in self.records.values():
                for i, p in enumerate(r.pages[gi]):
                    if p >= 0:
                        held.setdefault(p, []).append((i, (i + 1) * PAGE <= r.length))
            if len(held) != g.pool.in_use:
                raise CacheError(f"group {gi}: {g.pool.in_use} pages are out but sequences hold {len(held)}")
            for p, places in held.items():
                if len(places) != g.pool.holders(p):
                    raise CacheError(f"page {p} of group {gi} is held by {len(places)} sequences, the pool says {g.pool.holders(p)}")
                if len(places) > 1 and (len(set(places)) != 1 or not places[0][1]):
                    raise CacheError(f"a page of group {gi} is held by two sequences that may write to it")
        if set(self.records) != {i for i in range(self.max_slots) if self.slots._held[i]}:
            raise CacheError("open records and held slots differ")
