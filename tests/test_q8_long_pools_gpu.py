"""The cache in 8 bits behind offsets past 32 bits, and prompts captured into graphs."""
import pytest
import torch

from test_q8_gpu import BF, PAGE, Case, K  # noqa: F401
from test_q8_steps_gpu import tiles_of

pytestmark = pytest.mark.gpu


def moved(K, c, pools, exps, shift):
    """The case's pages as pages ``shift`` on of larger pools; returns the cache and the step."""
    small, _ = c.device(K)
    for big, t in zip((pools[0], exps[0], pools[1], exps[1]), small):
        big[shift:shift + c.pages].copy_(t)
    c.table = torch.where(c.table >= 0, c.table + shift, c.table)
    ints = [t for t in c.dev["ints"][:5]] + [c.table.cuda()]
    c.table = torch.where(c.table >= 0, c.table - shift, c.table)
    return (pools[0], exps[0], pools[1], exps[1]), K.step_batch(*ints)


def test_pages_past_4_gb(K):
    # 70,000 pages of 64 kB: the last of them begin at 4.6 GB
    kv, qpk, dim, pages = 8, 4, 128, 70000
    pools = [torch.zeros((pages, kv, PAGE, dim), dtype=torch.uint8, device="cuda").view(K.Q8) for _ in "kv"]
    exps = [torch.zeros((pages, kv), dtype=torch.int8, device="cuda") for _ in "kv"]
    results = []
    for shift in (0, pages - 60):
        got = []
        c = Case(kv, qpk, dim, [700, 64, 0], [1, 1, 1], rot=dim, seed=5)
        cache, batch = moved(K, c, pools, exps, shift)
        for splits in (1, 16):
            got.append(K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], None, kv, qpk, dim, c.scale, n_splits=splits))
        got += K.unpack_pages_q8(*cache, torch.arange(shift, shift + 10, dtype=torch.int32, device="cuda"))
        c = Case(kv, qpk, dim, [100, 0], [200, 130], rot=dim, seed=6)
        cache, batch = moved(K, c, pools, exps, shift)
        q = K.split_rotate_store_q8(c.dev["fused"], *cache, batch, kv, qpk, dim, rope=c.dev["rope"])
        lists, n_tiles = tiles_of(c.news, 128)
        for n_pages in (0, 8):
            got.append(K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, kv, c.scale, n_pages=n_pages))
        got += [cache[i][shift:shift + c.pages].view(torch.uint8).clone() for i in range(4)]
        K.copy_pages([p[None] for p in pools], [shift + 3], [shift + 50 if shift else pages - 5])
        got += [p[shift + 50 if shift else pages - 5].view(torch.uint8).clone() for p in pools]
        K.check_device_errors("cuda")
        results.append(got)
    for a, b in zip(*results):
        torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
    del pools, exps
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kv,qpk,dim,slopes", [(2, 4, 128, False), (1, 5, 64, True), (2, 2, 96, False)])
@pytest.mark.parametrize("unpacked", [True, False])
def test_prompts_captured_and_replayed_side_by_side(K, kv, qpk, dim, slopes, unpacked):
    c = Case(kv, qpk, dim, [300, 0], [200, 140], slopes=slopes, seed=9)
    q = c.split()[0].to(BF)
    c.append()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of(c.news, 128)
    qd = q.cuda()
    def call():
        return K.attention_q8(qd, *cache, batch, *lists, n_tiles, 128, c.dev["slopes"], kv, c.scale, n_pages=11 if unpacked else 0)
    first = call()
    c.check(first, q.float())
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(call())
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, graph in zip((side, other), graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    K.check_device_errors("cuda")
