"""Forks of long sequences (no GPU)."""
import time

import torch

from pytorch_transformers_b200.cache.paged import PAGE, Cache
from pytorch_transformers_b200.parts.base import CacheNeed


def test_a_copy_of_a_long_sequence_takes_time_by_its_pages():
    n = 60000      # with a walk over the copied pages for each page: ten seconds
    cache = Cache([(0, CacheNeed("full", 1, 1, v_head_dim=0), None)], (2 * n + 2) * PAGE, torch.bfloat16, "cpu")
    slot = cache.open()
    cache.reserve(slot, n * PAGE + 5)
    cache.commit(slot, n * PAGE + 5)
    t = time.perf_counter()
    new = cache.fork(slot, share=False)
    assert time.perf_counter() - t < 3.0
    assert cache.length(new) == n * PAGE + 5 and not set(cache.pages(new, 0)) & set(cache.pages(slot, 0))
    cache.check()
