"""Attention over a cache in 8 bits where more than a cluster of blocks shares a row's pages: the parts that join through memory."""
import ctypes

import pytest
import torch

from test_q8_gpu import BF, PAGE, Case, K  # noqa: F401

pytestmark = pytest.mark.gpu


# the rows of parts that no block has written: more splits than asked for by hand, and by the library's own choice behind a wide table
@pytest.mark.parametrize("splits,pages", [(16, 2), (24, 2), (0, 512)])
def test_a_step_without_one_token_each_writes_nothing(K, splits, pages):
    c = Case(1, 2, 64, [10, 20], [2, 0])
    cache, batch = c.device(K)
    before = [t.clone() for t in cache]
    guard = 6
    out = torch.full((2 + guard, 2 * 64), 7.0, dtype=BF, device="cuda")      # two rows of the result, and rows behind it
    L, stream = K.lib(), torch.cuda.current_stream().cuda_stream
    floats = L.ptb_attention_q8_floats(2, 1, 2, 1, 64, splits, pages, 2)
    assert floats > 0      # the parts join through memory
    parts = torch.full((floats,), 3.0, device="cuda")
    code = L.ptb_attention_decode_q8(c.dev["fused"].data_ptr(), *(t.data_ptr() for t in cache), c.pages, out.data_ptr(), ctypes.byref(batch), None,
                                     None, 0, False, None, 2, 1, 64, 0.1, 0, True, splits, pages, parts.data_ptr(), floats,
                                     K.error_flag("cuda").data_ptr(), stream)
    assert code == 0
    with pytest.raises(K.KernelError, match="one token for each"):
        K.check_device_errors("cuda")
    assert bool((out == 7.0).all())
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def tiles_of(news, tile):
    tiles = [(b, q0) for b, n in enumerate(news) for q0 in range(0, n, tile)]
    return [torch.tensor(x, dtype=torch.int32).cuda() for x in zip(*tiles)], len(tiles)


def floats(K, c, tiles, rows, tile, splits, pages):
    return K.lib().ptb_attention_q8_floats(tiles, c.kv, rows, tile, c.dim, splits, pages, sum(c.news))


@pytest.mark.parametrize("kv,qpk,dim", [(1, 3, 64), (2, 9, 128), (1, 40, 80), (1, 71, 64), (1, 100, 256)])
@pytest.mark.parametrize("pasts", [[9000], [9000, 0, 63, 700], [4095, 4096, 4097]])
@pytest.mark.parametrize("splits,window,slopes", [(16, 0, False), (24, 0, True), (64, 0, False), (512, 0, False), (16, 1000, False), (24, 65, True)])
def test_single_tokens(K, kv, qpk, dim, pasts, splits, window, slopes):
    # more blocks than a sequence has pages among them: those leave no weight
    c = Case(kv, qpk, dim, pasts, [1] * len(pasts), rot=0 if slopes else dim, slopes=slopes, window=window, seed=dim + splits)
    if window:
        c.give_back_left_of_windows()
    cache, batch = c.device(K)
    assert floats(K, c, len(pasts), qpk, 1, splits, 200) > 0
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], c.dev["slopes"], kv, qpk, dim, c.scale, window=window, n_splits=splits)
    c.append()
    c.check_cache()
    c.check(out, c.split()[0])
    K.check_device_errors("cuda")


def test_single_tokens_of_a_long_sequence_by_the_librarys_choice(K):
    c = Case(2, 4, 64, [16000, 200], [1, 1], rot=64, seed=3)
    cache, batch = c.device(K)
    assert floats(K, c, 2, 4, 1, 0, batch.pages_stride) > 0
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], None, 2, 4, 64, c.scale)
    c.append()
    c.check_cache()
    c.check(out, c.split()[0])
    K.check_device_errors("cuda")


@pytest.mark.parametrize("kv,qpk,dim", [(1, 3, 64), (2, 4, 128), (1, 17, 112), (1, 5, 256)])
@pytest.mark.parametrize("pasts,news,tile", [([8500], [17], 64), ([0, 4200, 64], [3, 40, 1], 64), ([3000, 0], [16, 5], 16), ([2000, 70], [130, 200], 128)])
@pytest.mark.parametrize("splits,window,slopes", [(16, 0, False), (24, 0, True), (32, 900, False)])
def test_chunks(K, kv, qpk, dim, pasts, news, tile, splits, window, slopes):
    c = Case(kv, qpk, dim, pasts, news, slopes=slopes, window=window, seed=dim + splits)
    if window:
        c.give_back_left_of_windows()
    q = c.split()[0].to(BF)
    c.append()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of(news, tile)
    assert floats(K, c, n_tiles, tile * qpk, tile, splits, batch.pages_stride) > 0
    out = K.attention_q8(q.cuda(), *cache, batch, *lists, n_tiles, tile, c.dev["slopes"], kv, c.scale, window=window, n_splits=splits)
    c.check(out, q.float())
    K.check_device_errors("cuda")


def test_a_chunk_after_a_long_past_by_the_librarys_choice(K):
    c = Case(1, 2, 64, [16500], [5], seed=3)
    q = c.split()[0].to(BF)
    c.append()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of([5], 16)
    assert floats(K, c, n_tiles, 32, 16, 0, batch.pages_stride) > 0
    out = K.attention_q8(q.cuda(), *cache, batch, *lists, n_tiles, 16, None, 1, c.scale)
    c.check(out, q.float())
    K.check_device_errors("cuda")


def test_captured_and_replayed_side_by_side(K):
    # two graphs of the same call, each with parts of its own
    c = Case(2, 4, 64, [5000, 700], [1, 1], seed=9)
    cache, batch = c.device(K)
    args = (c.dev["fused"], *cache, batch, None, None, 2, 4, 64, c.scale)
    first = K.attention_decode_q8(*args, n_splits=24)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(K.attention_decode_q8(*args, n_splits=24, write_cache=False))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, graph in zip((side, other), graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    K.check_device_errors("cuda")
