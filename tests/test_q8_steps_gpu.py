"""Prompts over a cache in 8 bits whose steps do not fit their page tables, and workspaces of steps."""
import pytest
import torch

from test_q8_gpu import BF, PAGE, Case, K  # noqa: F401

pytestmark = pytest.mark.gpu


def tiles_of(news, tile):
    tiles = [(b, q0) for b, n in enumerate(news) for q0 in range(0, n, tile)]
    return [torch.tensor(x, dtype=torch.int32).cuda() for x in zip(*tiles)], len(tiles)


@pytest.mark.parametrize("width", [0, 1, 2])
@pytest.mark.parametrize("kv,qpk,dim,slopes,window", [(1, 2, 64, False, 0), (1, 2, 128, False, 0), (2, 3, 128, True, 0), (1, 2, 64, True, 70), (1, 40, 128, False, 0),
                                                      (2, 2, 96, False, 0), (1, 2, 256, False, 0)])
@pytest.mark.parametrize("unpacked", [True, False])
def test_a_prompt_behind_a_table_too_narrow_is_said(K, kv, qpk, dim, slopes, window, width, unpacked):
    # sequences of one, two and eight pages behind a table of fewer: nothing past its rows is read, the others' results stand, and the
    # cache stays as it was
    c = Case(kv, qpk, dim, [20, 0, 300], [40, 128, 200], slopes=slopes, window=window, seed=3)
    q, _, _ = c.split()
    q = q.to(BF)
    whole = c.table
    c.append()
    c.table = whole[:, :width].contiguous()
    cache, batch = c.device(K)
    before = [t.clone() for t in cache]
    lists, n_tiles = tiles_of(c.news, 128)
    spans = 1 + 2 + 8 - (max(0, 300 - window + 1) // PAGE if window else 0)
    out = K.attention_q8(q.cuda(), *cache, batch, *lists, n_tiles, 128, c.dev["slopes"], kv, c.scale, window=window, n_pages=spans if unpacked else 0)
    with pytest.raises(K.KernelError, match="a page that the cache does not have"):
        K.check_device_errors("cuda")
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    if width:      # the sequence whose pages are all listed
        c.table = whole
        want, parts = c.attend(q.float())
        import plain_q8 as plain
        got = out.cpu().double().view(want.shape)[:40]
        assert bool(((got - want[:40]).abs() <= plain.bound(*parts[0])).all())


def test_descriptions_of_pools_that_come_and_go_are_not_kept_for_good(K):
    # the same pages as pools of 2,500 sizes: two descriptions each
    L = K.lib()
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(2600, 1, PAGE, 64, generator=g, device="cuda", dtype=BF) for _ in "kv")
    q = torch.randn(130, 2, 64, generator=g, device="cuda", dtype=BF)
    ints = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([0] * 130, list(range(130)), [0], [130], [0])]
    batch = K.step_batch(*ints, torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda())
    lists, n_tiles = tiles_of([130], 128)
    def run(pages):
        return K.attention_tc_extras(q, k[:pages], v[:pages], batch, *lists, n_tiles, 1, 0.125)
    first = run(3)
    for pages in range(4, 2504):
        run(pages)
    assert 0 < L.ptb_pool_maps() <= 2048
    assert torch.equal(run(3), first) and torch.equal(run(1000), first)
    K.check_device_errors("cuda")


def long_cache(K, kv, dim, tokens, seqs):
    """Pages of ``seqs`` sequences of ``tokens`` tokens, made on the device."""
    g = torch.Generator(device="cuda").manual_seed(0)
    per = (tokens + PAGE - 1) // PAGE
    cache = []
    for _ in "kv":
        cache += [torch.randn(seqs * per, kv, PAGE, dim, generator=g, device="cuda", dtype=BF).to(K.Q8), torch.zeros(seqs * per, kv, dtype=torch.int8, device="cuda")]
    return cache, torch.arange(seqs * per, dtype=torch.int32).view(seqs, per)


def described(K, table, pasts, news):
    ints = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([b for b, n in enumerate(news) for _ in range(n)],
                                                                [p + i for p, n in zip(pasts, news) for i in range(n)],
                                                                [sum(news[:b]) for b in range(len(news))], news, pasts)]
    return K.step_batch(*ints, table.cuda())


def test_a_prompt_beside_single_tokens_takes_no_workspace(K):
    # one of 32 sequences of 2,048 tokens brings 200, the others one each: their pages as bfloat16 values would be 268 MB
    pasts, news = [1800] + [2000] * 31, [200] + [1] * 31
    cache, table = long_cache(K, 8, 128, 2048, 32)
    batch = described(K, table, pasts, news)
    lists, n_tiles = tiles_of(news, 128)
    q = torch.randn(sum(news), 16, 128, device="cuda", dtype=BF)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 8, 0.1, n_pages=32 * 32)
    assert torch.cuda.max_memory_allocated() - before < 64 << 20
    assert torch.equal(out, K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 8, 0.1))
    K.check_device_errors("cuda")


def test_a_prompt_without_room_for_a_workspace_reads_the_codes(K):
    # 300 tokens after 60,000: pages of 247 MB as bfloat16 values, on a device that the process may not use more of
    cache, table = long_cache(K, 8, 128, 60300, 1)
    batch = described(K, table, [60000], [300])
    lists, n_tiles = tiles_of([300], 128)
    q = torch.randn(300, 16, 128, device="cuda", dtype=BF)
    want = K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 8, 0.1)
    pages = cache[0].shape[0]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            torch.empty(pages, 8, PAGE, 128, dtype=BF, device="cuda")
        out = K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 8, 0.1, n_pages=pages)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(out, want)
    K.check_device_errors("cuda")
    unpacked = K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 8, 0.1, n_pages=pages)
    # each off by its rounding (2^-8) and by weights of 11 bits beside values up to 5.5 (2^-11 of them)
    torch.testing.assert_close(unpacked.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


@pytest.mark.parametrize("window,width,n_pages", [(0, 2, 3), (70, 1, 1), (64, 2, 2), (500, 9, 4)])
def test_a_prompt_with_too_few_pages_behind_a_table_too_narrow_is_said(K, window, width, n_pages):
    c = Case(1, 2, 64, [300, 5, 300], [64, 130, 300], window=window, seed=3)
    q = c.split()[0].to(BF).cuda()
    c.append()
    whole, c.table = c.table, c.table[:, :width].contiguous()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of(c.news, 128)
    K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 1, c.scale, window=window, n_pages=n_pages)
    with pytest.raises(K.KernelError, match="page"):
        K.check_device_errors("cuda")
    c.table = whole      # and the next step is none the worse
    cache, batch = c.device(K)
    out = K.attention_q8(q, *cache, batch, *lists, n_tiles, 128, None, 1, c.scale, window=window, n_pages=24)
    c.check(out, q.cpu().float())
    K.check_device_errors("cuda")
