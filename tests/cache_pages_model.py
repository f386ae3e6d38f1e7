"""A cache under random forks, cuts, moves and steps beside lists of what every sequence holds."""
import random

import torch

from pytorch_transformers_b200.cache import PAGE, Cache, CacheError, CacheFull
from pytorch_transformers_b200.parts import CacheNeed, StateNeed


class Sequences:
    def __init__(self, device, dtype=torch.float32, kv_dtype=None, pages=24, window=0, state=0, max_slots=None, keep_first=0):
        needs = [CacheNeed("full", 2, 16, eight_bit=True), CacheNeed("window", 1, 32, window, keep_first=keep_first, eight_bit=True) if window
                 else CacheNeed("full", 2, 16, eight_bit=True)]
        self.cache = Cache([(0, needs[0], StateNeed(state) if state else None), (1, needs[1], None)], pages * PAGE, dtype, device,
                           max_slots=max_slots, kv_dtype=kv_dtype)
        self.held = {}       # slot -> token numbers
        self.next = 1
        self.state = state

    def numbers(self, n):
        out = list(range(self.next, self.next + n))
        self.next += n
        return out

    def _bytes(self, t, number):
        """What a token leaves in a row of tensor ``t``: bytes that follow from its number."""
        width = t.shape[-1] * t.element_size()
        return ((torch.arange(width) * 31 + number * 7 + number // 200) % 120).to(torch.uint8)

    def append(self, slot, n):
        self.cache.reserve_all([(slot, n)])
        tokens, past = self.numbers(n), self.cache.length(slot)
        for gi, g in enumerate(self.cache.groups):
            for i, number in enumerate(tokens):
                page, at = self.cache.pages(slot, gi)[(past + i) // PAGE], (past + i) % PAGE
                for t in (g.k, g.v):
                    t.view(torch.uint8)[:, page, :, at] = self._bytes(t, number).to(t.device)
                if g.k_exp is not None:
                    g.k_exp[:, page] = tokens[0] % 100       # the page's exponent: of its last writer
                    g.v_exp[:, page] = tokens[0] % 90
        if self.state:
            self.cache.state[slot] = float(tokens[-1])
        self.cache.commit(slot, n)
        self.held[slot].extend(tokens)

    def open(self):
        slot = self.cache.open()
        self.held[slot] = []
        return slot

    def fork(self, slot, share=True):
        new = self.cache.fork(slot, share=share)
        assert new not in self.held
        self.held[new] = list(self.held[slot])
        return new

    def close(self, slot):
        self.cache.close(slot)
        del self.held[slot]

    def truncate(self, slot, length):
        self.cache.truncate(slot, length)
        del self.held[slot][length:]

    def check(self):
        self.cache.check()
        for slot, tokens in self.held.items():
            assert self.cache.length(slot) == len(tokens)
            for gi, g in enumerate(self.cache.groups):
                pages = self.cache.pages(slot, gi)
                assert len(pages) * PAGE >= len(tokens)
                first = max(0, len(tokens) - g.need.window + 1) // PAGE * PAGE if g.need.kind == "window" else 0
                for t in (g.k, g.v):
                    raw = t.view(torch.uint8).cpu()
                    for i, number in enumerate(tokens):
                        if i < first and i >= g.need.keep_first:
                            continue
                        want = self._bytes(t, number)
                        assert torch.equal(raw[0, pages[i // PAGE], 0, i % PAGE], want)
                        assert torch.equal(raw[-1, pages[i // PAGE], -1, i % PAGE], want)
            if self.state and tokens:
                assert float(self.cache.state[slot, 0]) == tokens[-1]


def random_walk(s: Sequences, seed: int, steps: int, most=70):
    rng = random.Random(seed)
    for _ in range(steps):
        slots = list(s.held)
        what = rng.choice(["open", "append", "append", "fork", "fork", "close", "truncate", "compact", "resize"])
        before = ({k: list(v) for k, v in s.held.items()}, [g.pool.in_use for g in s.cache.groups])
        try:
            if what == "open":
                s.open()
            elif what == "compact":
                s.cache.compact()
                for g in s.cache.groups:
                    assert all(g.pool.holders(i) for i in range(g.pool.in_use))
            elif what == "resize":
                s.cache.resize(rng.choice([8, 16, 24, 40]) * PAGE - rng.randrange(64))
            elif slots:
                slot = rng.choice(slots)
                if what == "append":
                    s.append(slot, rng.choice([1, 1, 63, 64, 65, rng.randrange(1, most)]))
                elif what == "fork":
                    s.fork(slot, share=rng.random() < 0.8)
                elif what == "close":
                    s.close(slot)
                else:
                    s.truncate(slot, rng.randrange(len(s.held[slot]) + 1))
        except (CacheFull, CacheError):      # refused before anything changed
            assert before == ({k: list(v) for k, v in s.held.items()}, [g.pool.in_use for g in s.cache.groups])
        s.check()
