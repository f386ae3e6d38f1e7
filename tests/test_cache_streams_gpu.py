"""Caches whose pages move on another stream than the one that their storage was allocated on."""
import pytest
import torch

from pytorch_transformers_b200.cache.paged import PAGE, Cache
from pytorch_transformers_b200.parts.base import CacheNeed, StateNeed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_dtype", [None, torch.float8_e4m3fn])
def test_resize_on_another_stream_keeps_what_it_copies(kv_dtype):
    need = CacheNeed("full", 2, 64, eight_bit=True)
    cache = Cache([(0, need, StateNeed(40)), (1, need, None)], 100 * PAGE, torch.bfloat16, "cuda", kv_dtype=kv_dtype)
    slot = cache.open()
    cache.reserve(slot, 90 * PAGE)
    cache.commit(slot, 90 * PAGE)
    group = cache.groups[0]
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in group.tensors():
        t.view(torch.uint8).random_(0, 256, generator=g)
    cache.state.random_(0, 256, generator=g)
    want, state = [t.view(torch.uint8).clone() for t in group.tensors()], cache.state.clone()
    sizes = [(t.shape, t.dtype) for t in group.tensors() + [cache.state]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)      # a tenth of a second: the copies wait
        cache.resize(300 * PAGE)
    # tensors that would fit where the old storage was, written at once
    junk = [torch.full(shape, 3, dtype=torch.uint8 if dtype.itemsize == 1 else torch.int16 if dtype.itemsize == 2 else torch.int32, device="cuda")
            for shape, dtype in sizes * 3]
    torch.cuda.synchronize()
    for t, w in zip(group.tensors(), want):
        assert torch.equal(t.view(torch.uint8)[:, :90], w[:, :90])
    assert torch.equal(cache.state[:100], state)
    assert len(junk) == 3 * len(sizes)
    cache.check()
