"""The cache in 8 bits on the device: appending, reading back, attention of single tokens and of prompts, copies of pages,
each against a plain implementation in 64 bits (plain_q8)."""
import math

import numpy as np
import pytest
import torch

import plain_q8 as plain

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
PAGE = 64


@pytest.fixture(scope="module")
def K():
    from pytorch_transformers_b200 import kernels
    kernels.lib()
    return kernels


class Case:
    """A cache of one entry with sequences of ``pasts`` tokens, and the step that brings ``news`` more. The pages' rows that no token has
    written hold no numbers, and so do pages that no sequence holds."""

    def __init__(self, kv, qpk, dim, pasts, news, rot=0, interleaved=False, slopes=False, window=0, seed=0, spread=1.0, extra=2):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.qpk, self.dim, self.pasts, self.news, self.window = kv, qpk, dim, pasts, news, window
        self.heads, self.interleaved, self.scale = kv * qpk, interleaved, 1.0 / math.sqrt(dim)
        counts = [(p + n + PAGE - 1) // PAGE for p, n in zip(pasts, news)]
        self.pages = sum(counts) + extra
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((len(pasts), max(counts) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        tokens = sum(news)
        self.seq_of = [b for b, n in enumerate(news) for _ in range(n)]
        self.pos = [p + i for p, n in zip(pasts, news) for i in range(n)]
        self.start = [sum(news[:b]) for b in range(len(news))]
        shape = (self.pages, kv, PAGE, dim)
        self.codes, self.exps = {}, {}
        for name in "kv":
            self.codes[name] = torch.full(shape, math.nan, dtype=torch.float64)
            self.exps[name] = torch.randint(-9, 9, shape[:2], generator=g).to(torch.int8)
            for b, p in enumerate(pasts):
                for i in range((p + PAGE - 1) // PAGE):
                    rows = torch.randn(kv, min(PAGE, p - i * PAGE), dim, generator=g) * spread ** torch.randn(kv, 1, 1, generator=g)
                    plain.append(self.codes[name], self.exps[name], int(self.table[b, i]), 0, rows)
        self.fused = torch.randn(tokens, kv * (qpk + 2) * dim, generator=g).to(BF)
        self.cos = self.sin = None
        if rot:
            angle = torch.tensor(self.pos)[:, None] * (1.0 / 10000.0 ** (torch.arange(0, rot, 2) / rot))[None]
            self.cos, self.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        self.slopes = (2.0 ** (-8.0 * torch.arange(1, self.heads + 1) / self.heads)).bfloat16().float() if slopes else None

    def give_back_left_of_windows(self):
        for b, p in enumerate(self.pasts):
            self.table[b, :max(0, p - self.window + 1) // PAGE] = -1

    def device(self, K):
        """The same on the device: (k_pool, k_exp, v_pool, v_exp), batch."""
        d = self.dev = {}
        for name in "kv":
            d[name] = self.codes[name].float().to(K.Q8).cuda()
            d[name + "e"] = self.exps[name].cuda()
        def ints(x):
            return torch.as_tensor(x, dtype=torch.int32).cuda().contiguous()
        d["ints"] = [ints(x) for x in (self.seq_of, self.pos, self.start, self.news, self.pasts)] + [self.table.cuda()]
        d["fused"] = self.fused.cuda()
        d["rope"] = (self.cos.cuda(), self.sin.cuda()) if self.cos is not None else None
        d["slopes"] = self.slopes.cuda() if self.slopes is not None else None
        return (d["k"], d["ke"], d["v"], d["ve"]), K.step_batch(*d["ints"])

    def split(self):
        f = self.fused.float().view(-1, self.kv, self.qpk + 2, self.dim)
        q = plain.rotate(f[:, :, :self.qpk].reshape(-1, self.heads, self.dim), self.cos, self.sin, self.interleaved)
        return q, plain.rotate(f[:, :, self.qpk], self.cos, self.sin, self.interleaved), f[:, :, self.qpk + 1]

    def append(self):
        _, k, v = self.split()
        for b, (p, n) in enumerate(zip(self.pasts, self.news)):
            for i in range(p // PAGE, (p + n - 1) // PAGE + 1):
                lo, hi = max(p, i * PAGE), min(p + n, (i + 1) * PAGE)
                for name, x in (("k", k), ("v", v)):
                    rows = x[self.start[b] + lo - p:self.start[b] + hi - p].transpose(0, 1)
                    plain.append(self.codes[name], self.exps[name], int(self.table[b, i]), lo - i * PAGE, rows)

    def check_cache(self):
        for name in "kv":
            assert torch.equal(self.exps[name], self.dev[name + "e"].cpu()), name
            got = self.dev[name].float().cpu().double()
            torch.testing.assert_close(got, self.codes[name], rtol=0, atol=0, equal_nan=True)

    def attend(self, q):
        """(outputs, how far they may be off by seq and size) of queries [tokens, heads, dim]."""
        outs, parts = [], []
        for b, (p, n) in enumerate(zip(self.pasts, self.news)):
            if not n:
                continue
            count = (p + n + PAGE - 1) // PAGE
            ids = self.table[b, :count].long().clamp(min=0)
            k, v = (plain.values(self.codes[x], self.exps[x])[ids].transpose(1, 2).reshape(-1, self.kv, self.dim)[:p + n] for x in "kv")
            o = plain.attend(q[self.start[b]:self.start[b] + n], k, v, self.scale, torch.arange(p, p + n), self.slopes, self.window)
            outs.append(o[0])
            parts.append((*o, p + n))
        return torch.cat(outs), parts

    def check(self, got, q, **bits):
        out, parts = self.attend(q)
        limit = torch.cat([plain.bound(*p, **bits) for p in parts])
        got = got.cpu().double().view(out.shape)
        assert torch.isfinite(got).all()
        over = (got - out).abs() - limit
        assert float(over.max()) <= 0, f"off by {float((got - out).abs().flatten()[over.argmax()])}, allowed {float(limit.flatten()[over.argmax()])}"


SHAPES = [(1, 71, 64), (8, 4, 128), (2, 16, 64), (3, 1, 16), (2, 3, 80), (1, 128, 128), (2, 5, 256), (1, 20, 192), (2, 2, 48), (1, 17, 112)]
ROTATIONS = [(0, False), (1.0, False), (0.5, False), (1.0, True), (0.5, True)]      # share of the head


# ------------------------------------------------------------------------------------------------ appending
@pytest.mark.parametrize("kv,qpk,dim", SHAPES)
@pytest.mark.parametrize("share,interleaved", ROTATIONS)
@pytest.mark.parametrize("pasts,news", [([0, 0, 0], [1, 64, 131]), ([1, 63, 64, 100, 0], [1, 1, 1, 1, 1]), ([5, 120, 64, 0], [60, 9, 64, 200])])
def test_append(K, kv, qpk, dim, share, interleaved, pasts, news):
    c = Case(kv, qpk, dim, pasts, news, rot=int(dim * share) // 2 * 2, interleaved=interleaved, seed=kv + dim, spread=4.0)
    cache, batch = c.device(K)
    q = K.split_rotate_store_q8(c.dev["fused"], *cache, batch, kv, qpk, dim, rope=c.dev["rope"], interleaved=interleaved)
    c.append()
    c.check_cache()
    assert torch.equal(q.cpu(), c.split()[0].to(BF))
    K.check_device_errors(q.device)


@pytest.mark.parametrize("rot", [2, 10, 20, 46])
def test_append_rotations_of_odd_widths(K, rot):
    c = Case(2, 3, 48, [0, 70], [70, 3], rot=rot, seed=rot)
    cache, batch = c.device(K)
    q = K.split_rotate_store_q8(c.dev["fused"], *cache, batch, 2, 3, 48, rope=c.dev["rope"])
    c.append()
    c.check_cache()
    assert torch.equal(q.cpu(), c.split()[0].to(BF))


@pytest.mark.parametrize("kind", ["zero", "tiny", "huge", "inf", "nan", "all nan", "steps"])
def test_append_odd_numbers(K, kind):
    c = Case(2, 2, 32, [0, 40], [30, 24], seed=7)
    f = c.fused.view(-1, 2, 4, 32)
    if kind == "zero":
        f[:, :, 2:] = 0
    elif kind == "tiny":
        f[:, :, 2:] *= 2.0 ** -130
    elif kind == "huge":
        f[:, :, 2:] = torch.sign(f[:, :, 2:]) * 3.38e38
    elif kind == "inf":
        f[3, :, 2, 5], f[40, :, 3, 7] = math.inf, -math.inf
    elif kind == "nan":
        f[3, :, 2, 5], f[40, :, 3, 7] = math.nan, math.nan
    elif kind == "all nan":
        f[:, :, 2:] = math.nan
    else:      # exactly between two codes, at the largest code and next to it
        f[:, :, 2:] = torch.tensor([448.0, 1.0625, 1.1875, 0.0009765625, 0.0029296875, 432.0, -17.0, 2.0 ** -10]).repeat(4)
    cache, batch = c.device(K)
    K.split_rotate_store_q8(c.dev["fused"], *cache, batch, 2, 2, 32)
    c.append()
    c.check_cache()


def test_append_token_by_token_raises_exponents(K):
    # rows that grow by 1.7 a token: exponents rise again and again, and every earlier code is rounded each time
    c = Case(1, 1, 64, [0], [70], seed=3)
    c.fused = (torch.randn(70, 192, generator=torch.Generator().manual_seed(1)) * 1.7 ** torch.arange(70)[:, None]).to(BF)
    whole, news = c.fused, []
    cache, _ = c.device(K)
    for t in range(70):
        step = Case(1, 1, 64, [t], [1])
        step.fused, step.table, step.codes, step.exps, step.pages = whole[t:t + 1], c.table, c.codes, c.exps, c.pages
        step.append()
        ints = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([0], [t], [0], [1], [t])]
        table = c.table.cuda()
        out = K.attention_decode_q8(step.fused.cuda(), *cache, K.step_batch(*ints, table), None, None, 1, 1, 64, 0.125)
        news.append(out)
    c.check_cache()


def test_write_cache_false_leaves_the_cache_alone(K):
    c = Case(2, 3, 64, [10, 64, 0], [1, 1, 1], rot=64)
    cache, batch = c.device(K)
    K.split_rotate_store_q8(c.dev["fused"], *cache, batch, 2, 3, 64, rope=c.dev["rope"], write_cache=False)
    c.check_cache()


# ------------------------------------------------------------------------------------------------ reading back
@pytest.mark.parametrize("kv,dim", [(1, 64), (8, 128), (3, 80), (2, 256), (5, 16)])
def test_unpack(K, kv, dim):
    c = Case(kv, 1, dim, [200, 64], [1, 1], spread=30.0)
    cache, _ = c.device(K)
    ids = torch.tensor([c.pages - 1, 0, 2, 0], dtype=torch.int32).cuda()
    for name, got in zip("kv", K.unpack_pages_q8(*cache, ids)):
        want = plain.values(c.codes[name], c.exps[name])[ids.cpu().long()]
        torch.testing.assert_close(got.cpu().double(), want, rtol=0, atol=0, equal_nan=True)
    K.check_device_errors(ids.device)


# ------------------------------------------------------------------------------------------------ single tokens
@pytest.mark.parametrize("kv,qpk,dim", SHAPES)
@pytest.mark.parametrize("position", ["half", "pairs", "alibi", "none"])
@pytest.mark.parametrize("splits", [0, 1, 3, 11])
def test_decode(K, kv, qpk, dim, position, splits):
    pasts = [0, 1, 15, 16, 62, 63, 64, 65, 200, 700]
    c = Case(kv, qpk, dim, pasts, [1] * len(pasts), rot=dim if position in ("half", "pairs") else 0, interleaved=position == "pairs",
             slopes=position == "alibi", seed=dim + splits, spread=2.0)
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], c.dev["slopes"], kv, qpk, dim, c.scale,
                                interleaved=c.interleaved, n_splits=splits)
    c.append()
    c.check_cache()
    c.check(out, c.split()[0])
    K.check_device_errors(out.device)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("kv,qpk,dim,splits", [(2, 3, 64, 0), (1, 40, 128, 2), (2, 2, 80, 1)])
@pytest.mark.parametrize("slopes", [False, True])
def test_decode_window(K, kv, qpk, dim, splits, window, slopes):
    c = Case(kv, qpk, dim, [0, 63, 64, 300, 127, 513], [1] * 6, slopes=slopes, window=window, seed=window)
    c.give_back_left_of_windows()
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, c.dev["slopes"], kv, qpk, dim, c.scale, window=window,
                                n_splits=splits)
    c.append()
    c.check_cache()
    c.check(out, c.split()[0])
    K.check_device_errors(out.device)


def test_decode_most_rows_of_the_widest_heads(K):
    c = Case(1, 128, 256, [70, 3], [1, 1], rot=256, seed=12)
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], None, 1, 128, 256, c.scale)
    c.append()
    c.check_cache()
    c.check(out, c.split()[0])


def test_decode_many_tiles_a_warp(K):
    # one block for 9,000 keys: a warp looks pages up in stretches of 32 tiles
    c = Case(1, 3, 64, [9000, 4097, 32 * 16 * 8 - 1], [1, 1, 1], seed=11)
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 3, 64, c.scale, n_splits=1)
    c.append()
    c.check(out, c.split()[0])


@pytest.mark.parametrize("exps", [(0, 60, -60), (-120, 100, 0, -126, 119), (5, -80, -80, 5), (119, -126, 119)])
def test_decode_pages_of_very_different_sizes(K, exps):
    # values' exponents far apart; weights about even, so that the largest page decides, as it does in 64 bits
    c = Case(2, 2, 64, [64 * len(exps) - 10], [1], seed=2)
    for i, e in enumerate(exps):
        c.exps["v"][int(c.table[0, i])] = e
    c.fused.view(1, 2, 4, 64)[:, :, 3] *= 2.0 ** max(-100, exps[-1])
    cache, batch = c.device(K)
    for splits in (1, 2):
        keep = [t.clone() for t in cache]
        out = K.attention_decode_q8(c.dev["fused"], *keep, batch, None, None, 2, 2, 64, c.scale, n_splits=splits)
        if splits == 1:
            c.append()
        c.check(out, c.split()[0])


def small_after_large(low):
    c = Case(1, 1, 64, [120], [1], seed=4)
    c.codes["k"][int(c.table[0, 0]), :, :, 0] = -448.0
    c.exps["k"][int(c.table[0, 0])] = 2
    c.exps["v"][int(c.table[0, 0])] = 10
    c.exps["v"][int(c.table[0, 1])] = low
    c.fused.view(1, 1, 3, 64)[:, :, 0, 0] = 4.0
    c.fused.view(1, 1, 3, 64)[:, :, 2] *= 2.0 ** low
    return c


@pytest.mark.parametrize("low", [-20, -55])
def test_decode_large_scores_either_way(K, low):
    # scores of some hundreds: the page of large values has the largest of them
    c = small_after_large(low)
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 1, 64, c.scale, n_splits=1)
    c.append()
    c.check(out, c.split()[0])


@pytest.mark.parametrize("low", [-20, -55])
def test_decode_small_values_seen_after_large_ones(K, low):
    # the weights leave out the page of large values (its keys point away from the query), so the output is that of the small page
    c = small_after_large(low)
    c.codes["k"][int(c.table[0, 0]), :, :, 1:] = 0.0
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 1, 64, c.scale, n_splits=1)
    c.append()
    want, parts = c.attend(c.split()[0])
    assert float(want.abs().max()) < 2.0 ** (low + 10)
    # the weights of the large page are below 2^-1000: the values that a row sees are the small page's
    _, _, size, keys = parts[0]
    most = c.codes["v"][int(c.table[0, 1]), :, :57].abs().amax().reshape(1, 1) * 2.0 ** low
    small = torch.nan_to_num(plain.values(c.codes["k"], c.exps["k"])[int(c.table[0, 1])]).abs().amax() * 64 * 5 * c.scale
    limit = plain.bound(want, most, torch.minimum(size, small.reshape(1, 1)), keys)
    assert bool(((out.cpu().double().view(want.shape) - want).abs() <= limit).all())


@pytest.mark.parametrize("splits", [1, 3])
def test_decode_no_numbers_reach_their_row_only(K, splits):
    c = Case(1, 4, 64, [150, 150], [1, 1], seed=5)
    c.codes["v"][int(c.table[0, 1]), 0, 3, 7] = math.nan
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 4, 64, c.scale, n_splits=splits).view(2, 4, 64)
    assert torch.isnan(out[0, :, 7]).all() and torch.isfinite(out[0, :, :7]).all() and torch.isfinite(out[1]).all()


def test_decode_reads_a_row_that_the_cache_holds(K):
    c = Case(2, 3, 64, [10, 64, 500], [1, 1, 1], rot=64)
    cache, batch = c.device(K)
    a = K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], None, 2, 3, 64, c.scale)
    c.append()
    b = K.attention_decode_q8(c.dev["fused"], *cache, batch, c.dev["rope"], None, 2, 3, 64, c.scale, write_cache=False)
    assert torch.equal(a, b)
    c.check_cache()


def test_decode_is_the_same_alone_and_in_a_batch(K):
    c = Case(2, 4, 64, [100, 700, 31], [1, 1, 1], seed=8)
    cache, batch = c.device(K)
    whole = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 2, 4, 64, c.scale, n_splits=2)
    for b in range(3):
        ints = [torch.tensor([x], dtype=torch.int32).cuda() for x in (0, c.pasts[b], 0, 1, c.pasts[b])]
        table = c.dev["ints"][5][b:b + 1].contiguous()
        one = K.attention_decode_q8(c.dev["fused"][b:b + 1].contiguous(), *cache, K.step_batch(*ints, table), None, None, 2, 4, 64, c.scale,
                                    n_splits=2)
        assert torch.equal(one[0], whole[b])


# ------------------------------------------------------------------------------------------------ prompts
def run_prompt(K, c, n_pages, tile=None):
    from pytorch_transformers_b200.parts.attention import AttentionTiles
    longest = max(c.news)
    tile = tile or (16 if longest <= 16 else 64 if longest <= 64 else 128)
    tiles = [(b, q0) for b, n in enumerate(c.news) for q0 in range(0, n, tile)]
    lists = [torch.tensor(x, dtype=torch.int32).cuda() for x in zip(*tiles)]
    cache, batch = c.device(K)
    q = K.split_rotate_store_q8(c.dev["fused"], *cache, batch, c.kv, c.qpk, c.dim, rope=c.dev["rope"], interleaved=c.interleaved)
    out = K.attention_q8(q, *cache, batch, *lists, len(tiles), tile, c.dev["slopes"], c.kv, c.scale, window=c.window, n_pages=n_pages)
    c.append()
    c.check_cache()
    K.check_device_errors(q.device)
    return out, q.cpu().float()


@pytest.mark.parametrize("kv,qpk,dim", SHAPES)
@pytest.mark.parametrize("pasts,news", [([0, 0], [2, 16]), ([100, 0, 63], [5, 16, 1]), ([0, 700], [40, 64]), ([0, 33, 300], [131, 200, 3])])
@pytest.mark.parametrize("position", ["half", "alibi"])
def test_prompts(K, kv, qpk, dim, pasts, news, position):
    c = Case(kv, qpk, dim, pasts, news, rot=dim if position == "half" else 0, slopes=position == "alibi", seed=dim, spread=2.0)
    out, q = run_prompt(K, c, 0)
    c.check(out, q)


@pytest.mark.parametrize("window", [1, 16, 63, 64, 100, 150])
@pytest.mark.parametrize("kv,qpk,dim", [(2, 3, 64), (1, 9, 80), (2, 2, 128)])
@pytest.mark.parametrize("pages", [0, 1])
def test_prompts_window(K, kv, qpk, dim, window, pages):
    for pasts, news in (([0, 300], [150, 129]), ([200, 64], [30, 64])):
        c = Case(kv, qpk, dim, pasts, news, window=window, seed=window)
        c.give_back_left_of_windows()
        out, q = run_prompt(K, c, pages * sum((p + n + PAGE - 1) // PAGE for p, n in zip(pasts, news)))
        c.check(out, q)


@pytest.mark.parametrize("kv,qpk,dim", [(1, 5, 64), (2, 4, 128), (3, 1, 64)])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("pasts,news", [([0], [129]), ([70, 0, 500], [200, 2, 140]), ([0, 64], [300, 128])])
def test_prompts_unpacked(K, kv, qpk, dim, slopes, pasts, news):
    # tiles of 128 tokens with the pages' number given: pages as bfloat16 values, then the tcgen05 kernel; with slopes its
    # weights are bfloat16 numbers of 8 bits (their rounding and the sum of the unrounded ones: twice)
    c = Case(kv, qpk, dim, pasts, news, slopes=slopes, seed=dim + qpk)
    out, q = run_prompt(K, c, sum((p + n + PAGE - 1) // PAGE for p, n in zip(pasts, news)) + 1, tile=128)
    c.check(out, q, weight_bits=7 if slopes else 11)


@pytest.mark.parametrize("kv,qpk,dim", [(1, 5, 16), (2, 3, 48), (3, 2, 96), (1, 7, 112), (2, 2, 64), (1, 4, 128)])
@pytest.mark.parametrize("slopes,window", [(False, 0), (True, 0), (False, 130), (True, 130)])
def test_prompts_unpacked_of_other_heads(K, kv, qpk, dim, slopes, window):
    # heads that the prompt kernel takes as 64 or 128 entries, and slopes beside a window; weights of two terms throughout
    pasts, news = [0, 300, 64], [131, 200, 3]
    c = Case(kv, qpk, dim, pasts, news, slopes=slopes, window=window, seed=dim + qpk, spread=2.0)
    if window:
        c.give_back_left_of_windows()
    out, q = run_prompt(K, c, sum((p + n + PAGE - 1) // PAGE for p, n in zip(pasts, news)))
    c.check(out, q)


# ------------------------------------------------------------------------------------------------ graphs and streams
def test_captured_and_replayed_on_another_stream(K):
    c = Case(2, 4, 64, [100, 2000], [1, 1], rot=64, seed=9)
    cache, batch = c.device(K)
    args = (c.dev["fused"], *cache, batch, c.dev["rope"], None, 2, 4, 64, c.scale)
    first = K.attention_decode_q8(*args, n_splits=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(K.attention_decode_q8(*args, n_splits=3, write_cache=False))
        graphs.append(graph)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):      # two graphs of the same call side by side: they share no workspace
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)


# ------------------------------------------------------------------------------------------------ copies
@pytest.mark.parametrize("shape,dtype", [((3, 20, 2, 64, 80), BF), ((2, 30, 1, 64, 64), torch.float32), ((4, 25, 3), torch.int8),
                                         ((2, 40, 8, 64, 128), torch.float8_e4m3fn), ((1, 9, 5, 7, 3), torch.int16), ((2, 11, 3), torch.float32)])
def test_copy_pages(K, shape, dtype):
    g = torch.Generator().manual_seed(1)
    pools = [torch.randint(0, 255, shape[:-1] + (shape[-1] * torch.empty((), dtype=dtype).element_size(),), generator=g,
                           dtype=torch.uint8).cuda().view(dtype) for _ in range(2)]
    before = [p.clone() for p in pools]
    order = torch.randperm(shape[1], generator=g)
    n = shape[1] // 2
    src, dst = order[:n].numpy(), order[n:2 * n].numpy()
    src[1:3] = src[0]      # a source for several targets
    def raw(t):
        return t.view(torch.uint8)
    assert K.copy_pages(pools, src, dst)[0] is pools[0]
    for a, b in zip(pools, before):
        want = raw(b).clone()
        want[:, torch.from_numpy(dst)] = raw(b)[:, torch.from_numpy(src)]
        assert torch.equal(raw(a), want)
    # into other storage with more pages, targets that are numbers of sources too
    others = [torch.zeros((shape[0], shape[1] + 5) + shape[2:], dtype=torch.uint8).cuda() if dtype == torch.uint8 else
              torch.zeros((shape[0], shape[1] + 5) + tuple(shape[2:]), device="cuda").to(dtype) for _ in range(2)]
    K.copy_pages(before, list(range(shape[1])), list(range(5, shape[1] + 5)), out=others)
    for a, b in zip(others, before):
        assert torch.equal(raw(a)[:, 5:], raw(b)) and not raw(a)[:, :5].any()


def test_copy_of_thousands_of_pages(K):
    pool = torch.arange(5000 * 6, dtype=torch.int32).view(1, 5000, 6).cuda()
    want = pool.clone()
    src, dst = np.arange(2500), np.arange(2500, 5000)[::-1]
    want[:, torch.from_numpy(dst.copy())] = want[:, torch.from_numpy(src)]
    K.copy_pages([pool], src, dst)
    assert torch.equal(pool, want)


@pytest.mark.parametrize("src,dst", [([0, 1], [2, 2]), ([0], [20]), ([-1], [3]), ([0, 1], [1, 2]), ([20], [0]), ([3], [3])])
def test_copy_refuses(K, src, dst):
    pool = torch.zeros(2, 20, 4).cuda()
    with pytest.raises(K.KernelError, match="page"):
        K.copy_pages([pool], src, dst)
    with pytest.raises(K.KernelError):
        K.copy_pages([pool], [0], [0], out=[pool[:, :, :]])
    with pytest.raises(K.KernelError):
        K.copy_pages([pool], [0, 1], [2])
    with pytest.raises(K.KernelError):
        K.copy_pages([pool], [0], [1], out=[torch.zeros(2, 20, 5).cuda()])


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(K):
    c = Case(2, 3, 64, [10], [1])
    (k, ke, v, ve), batch = c.device(K)
    f = c.dev["fused"]
    err = pytest.raises(K.KernelError)
    for bad in [(k.view(torch.uint8), ke, v, ve), (k, ke.float(), v, ve), (k, ke, v[:, :1], ve), (k, ke, v[:2], ve[:2]), (k, ke[:2], v, ve),
                (k.transpose(2, 3), ke, v, ve), (k.cpu(), ke, v, ve)]:
        with err:
            K.split_rotate_store_q8(f, *bad, batch, 2, 3, 64)
        with err:
            K.attention_decode_q8(f, *bad, batch, None, None, 2, 3, 64, 0.1)
    ok = (k, ke, v, ve)
    with err:
        K.attention_decode_q8(f.float(), *ok, batch, None, None, 2, 3, 64, 0.1)
    with err:
        K.attention_decode_q8(f[:, :-8], *ok, batch, None, None, 2, 3, 64, 0.1)
    with err:
        K.attention_decode_q8(f, *ok, batch, (torch.zeros(1, 33).cuda(),) * 2, None, 2, 3, 64, 0.1)
    with err:
        K.attention_decode_q8(f, *ok, batch, None, torch.zeros(5).cuda(), 2, 3, 64, 0.1)
    with err:
        K.attention_decode_q8(f, *ok, batch, None, None, 2, 3, 64, 0.1, window=-1)
    many = Case(1, 129, 16, [3], [1])
    cache, b2 = many.device(K)
    with err:
        K.attention_decode_q8(many.dev["fused"], *cache, b2, None, None, 1, 129, 16, 0.1)
    odd = Case(1, 2, 24, [3], [1])
    cache, b3 = odd.device(K)
    with err:
        K.attention_decode_q8(odd.dev["fused"], *cache, b3, None, None, 1, 2, 24, 0.1)
    two = Case(1, 2, 32, [3], [2])
    cache, b4 = two.device(K)
    with err:
        K.attention_decode_q8(two.dev["fused"], *cache, b4, None, None, 1, 2, 32, 0.1)


def test_a_page_that_does_not_exist_is_said(K):
    # the kernels check every page number of the table against the pool's size and read page 0 in its place
    for bad in (-1, 10 ** 6):
        c = Case(1, 2, 64, [100], [1])
        c.table[0, 0] = bad
        cache, batch = c.device(K)
        out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 2, 64, 0.1)
        with pytest.raises(K.KernelError):
            K.check_device_errors(out.device)
        ids = torch.tensor([0, bad], dtype=torch.int32).cuda()
        k, _ = K.unpack_pages_q8(*cache, ids)
        assert not k[1].any()
        with pytest.raises(K.KernelError):
            K.check_device_errors(out.device)


def test_as_many_tokens_as_sequences_but_not_one_each_is_said(K):
    c = Case(1, 2, 64, [10, 20], [2, 0])
    cache, batch = c.device(K)
    for call in (lambda: K.split_rotate_store_q8(c.dev["fused"], *cache, batch, 1, 2, 64),
                 lambda: K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 2, 64, 0.1)):
        call()
        with pytest.raises(K.KernelError, match="one token for each"):
            K.check_device_errors("cuda")


def test_fewer_pages_than_a_step_spans_are_said(K):
    for short, said in ((0, False), (1, True)):
        c = Case(1, 2, 64, [100, 0], [130, 200])
        cache, batch = c.device(K)
        q = torch.zeros(330, 2, 64, dtype=BF).cuda()
        lists = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 0, 1, 1], [0, 128, 0, 128])]
        K.attention_q8(q, *cache, batch, *lists, 4, 128, None, 1, 0.1, n_pages=4 + 4 - short)
        if said:
            with pytest.raises(K.KernelError, match="more pages than n_pages"):
                K.check_device_errors("cuda")
        else:
            K.check_device_errors("cuda")


def test_a_table_too_narrow_for_its_sequence_is_said(K):
    # two sequences of two and three pages behind a table one page wide: nothing past its rows is read, and only page 0, which the
    # missing ones read as, may be part of the result; the cache stays as it was
    c = Case(1, 2, 64, [100, 140], [1, 1])
    c.table = c.table[:, :1].contiguous()
    cache, batch = c.device(K)
    before = [t.clone() for t in cache]
    for call in (lambda: K.split_rotate_store_q8(c.dev["fused"], *cache, batch, 1, 2, 64),
                 lambda: K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 1, 2, 64, 0.1)):
        call()
        with pytest.raises(K.KernelError, match="page"):
            K.check_device_errors("cuda")
        for a, b in zip(cache, before):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
