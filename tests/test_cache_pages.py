"""Sequences forked, cut, moved and given back: nothing lost, nothing written that another sequence holds (no GPU)."""
import pytest
import torch

from cache_pages_model import Sequences, random_walk
from pytorch_transformers_b200.cache import PAGE, Cache, CacheError, CacheFull, IdPool
from pytorch_transformers_b200.modeling import resolve_cache_dtype
from pytorch_transformers_b200.parts import CacheNeed


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("kw", [dict(), dict(window=100), dict(window=40, keep_first=5), dict(state=3),
                                dict(dtype=torch.bfloat16, kv_dtype=torch.float8_e4m3fn, max_slots=5)], ids=str)
def test_random_walks(seed, kw):
    random_walk(Sequences("cpu", **kw), seed, 60)


def test_a_fork_shares_whole_pages_and_copies_the_last():
    s = Sequences("cpu", pages=8)
    a = s.open()
    s.append(a, 150)
    b = s.fork(a)
    for gi, g in enumerate(s.cache.groups):
        pa, pb = s.cache.pages(a, gi), s.cache.pages(b, gi)
        assert pa[:2] == pb[:2] and pa[2] != pb[2] and g.pool.in_use == 4
    s.append(a, 3)
    s.append(b, 50)
    s.check()
    s.close(a)
    s.check()
    assert s.cache.groups[0].pool.in_use == 4       # b's: two whole ones, its third and a fourth
    s.close(b)
    assert s.cache.groups[0].pool.in_use == 0


def test_a_fork_of_an_empty_and_of_a_full_page():
    s = Sequences("cpu", pages=4)
    a = s.open()
    s.cache.reserve(a, 200)                          # reserved ahead: the fork gets none of it
    b = s.fork(a)
    assert s.cache.pages(b, 0) == []
    s.truncate(a, 0)
    s.append(a, PAGE)
    c = s.fork(a)
    assert s.cache.pages(c, 0) == s.cache.pages(a, 0) and s.cache.groups[0].pool.in_use == 1
    s.append(c, 1)
    s.check()


def test_a_fork_without_room_changes_nothing():
    s = Sequences("cpu", pages=2)
    a = s.open()
    s.append(a, 100)
    epoch = s.cache.epoch
    with pytest.raises(CacheFull, match="fork needs 1 more"):
        s.fork(a)
    assert s.cache.epoch == epoch
    s.check()
    one = Sequences("cpu", pages=4, max_slots=1)
    a = one.open()
    one.append(a, 10)
    with pytest.raises(CacheFull):
        one.fork(a)
    one.check()


def test_cutting_into_a_shared_page_takes_one_of_its_own():
    s = Sequences("cpu", pages=3)
    a = s.open()
    s.append(a, 128)
    b = s.fork(a)
    s.truncate(b, 100)
    assert s.cache.pages(a, 0)[1] != s.cache.pages(b, 0)[1]
    s.append(b, 20)
    s.check()
    full = Sequences("cpu", pages=2)
    a = full.open()
    full.append(a, 128)
    b = full.fork(a)
    with pytest.raises(CacheFull, match="page of its own"):
        full.truncate(b, 100)
    full.truncate(b, 64)
    full.check()


def test_what_cannot_be_cut():
    s = Sequences("cpu", window=70)
    a = s.open()
    s.append(a, 300)
    with pytest.raises(CacheError, match="given back"):
        s.truncate(a, 150)
    with pytest.raises(ValueError):
        s.truncate(a, 301)
    with pytest.raises(ValueError):
        s.truncate(a, -1)
    with pytest.raises(CacheError, match="not open"):
        s.cache.truncate(17, 0)
    with pytest.raises(CacheError, match="not open"):
        s.cache.fork(17)
    t = Sequences("cpu", state=2)
    a = t.open()
    t.append(a, 10)
    with pytest.raises(CacheError, match="forget"):
        t.truncate(a, 5)
    t.cache.truncate(a, 10)


def test_resize_grows_slots_and_refuses_too_few_pages():
    s = Sequences("cpu", pages=3, state=1)
    a = s.open()
    s.append(a, 130)
    with pytest.raises(CacheFull, match="3 cache pages"):
        s.cache.resize(128)
    s.cache.resize(640)
    assert s.cache.num_pages == 10 and s.cache.max_slots == 10 and s.cache.groups[0].k.shape[1] == 10
    s.check()
    with pytest.raises(ValueError):
        s.cache.resize(0)


def test_captured_steps_are_dropped_with_the_storage():
    s = Sequences("cpu")
    s.cache.__dict__["_step_graphs"], s.cache.__dict__["_prepared_step"] = {1: 2}, (1, 2, 3)
    s.cache.resize(640)
    assert "_step_graphs" not in s.cache.__dict__ and "_prepared_step" not in s.cache.__dict__


def test_shared_ids():
    p = IdPool(3, "page")
    a, b = p.take(2)
    p.share([a])
    p.give_back([a])
    assert p.in_use == 2 and p.holders(a) == 1
    p.give_back([a])
    with pytest.raises(CacheError, match="freed twice"):
        p.give_back([a])
    with pytest.raises(CacheError, match="freed twice"):
        p.share([a])
    with pytest.raises(CacheError, match="outside"):
        p.share([3])
    assert p.renumber(3) == {b: a} and p.take(2) == [1, 2]
    with pytest.raises(CacheFull):
        p.renumber(2)
    p.check()


def test_which_caches_hold_8_bits():
    need = CacheNeed("full", 2, 16, eight_bit=True)
    f8 = torch.float8_e4m3fn
    c = Cache([(0, need, None)], 640, torch.bfloat16, "cpu", kv_dtype=f8)
    assert c.groups[0].k.dtype == f8 and c.groups[0].k_exp.shape == (1, 10, 2) and c.entry_exponents(0)[0].shape == (10, 2)
    assert c.groups[0].bytes() == 10 * 2 * 2 * (64 * 16 + 1)
    plain = Cache([(0, need, None)], 640, torch.bfloat16, "cpu", kv_dtype=torch.bfloat16)
    assert plain.kv_dtype is None and plain.entry_exponents(0) is None
    with pytest.raises(ValueError, match="8 bits"):
        Cache([(0, CacheNeed("full", 2, 16), None)], 640, torch.bfloat16, "cpu", kv_dtype=f8)
    for dtype, kv in ((torch.float32, f8), (torch.bfloat16, torch.int8), (torch.float32, torch.bfloat16)):
        with pytest.raises(ValueError):
            Cache([(0, need, None)], 640, dtype, "cpu", kv_dtype=kv)
    assert resolve_cache_dtype(None, torch.float32) is None and resolve_cache_dtype("bfloat16", torch.bfloat16) is None
    assert resolve_cache_dtype("float8_e4m3fn", torch.bfloat16) == f8
    with pytest.raises(ValueError):
        resolve_cache_dtype("int4", torch.bfloat16)


def test_a_resize_without_memory_for_the_second_group_leaves_what_is_held(monkeypatch):
    needs = [(0, CacheNeed("full", 1, 8), None), (1, CacheNeed("window", 1, 8, 100), None)]
    cache = Cache(needs, 6 * PAGE, torch.float32, "cpu")
    other = cache.open()
    slot = cache.open()
    for s in (other, slot):
        cache.reserve(s, 130)
        cache.commit(s, 130)
    for g in cache.groups:
        for i, p in enumerate(cache.pages(slot, cache.groups.index(g))):
            if p >= 0:
                g.k[:, p] = i + 1
    cache.close(other)                   # the lowest pages are free: those that are held will move
    epoch = cache.epoch
    with monkeypatch.context() as m:
        m.setattr(cache.groups[1], "_storage", lambda n: (_ for _ in ()).throw(MemoryError("none")))
        with pytest.raises(MemoryError):
            cache.resize(20 * PAGE)
    assert cache.epoch > epoch           # the first group's pages have moved: what was prepared for the old ones is stale
    cache.check()
    cache.resize(20 * PAGE)
    cache.check()
    for gi, g in enumerate(cache.groups):
        assert g.pool.capacity == 20
        for i, p in enumerate(cache.pages(slot, gi)):
            assert p < 0 or bool((g.k[:, p] == i + 1).all())
