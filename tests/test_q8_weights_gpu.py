"""Softmax weights of the attention over a cache in 8 bits: keys far below the largest score, as beside an attention sink, keep their
share of the output; pages whose values differ by large powers of two."""
import math

import pytest
import torch

import plain_q8 as plain
from test_q8_gpu import BF, PAGE, Case, K  # noqa: F401
from test_q8_steps_gpu import tiles_of

pytestmark = pytest.mark.gpu


def refill(c, b, k_rows, v_rows):
    """The pages of sequence ``b`` hold these rows [kv, tokens, dim] instead."""
    for name, rows in (("k", k_rows), ("v", v_rows)):
        for i in range((rows.shape[1] + PAGE - 1) // PAGE):
            plain.append(c.codes[name], c.exps[name], int(c.table[b, i]), 0, rows[:, i * PAGE:(i + 1) * PAGE])


def beside_a_sink(kv, qpk, dim, past, new, above, at, uneven=False, window=0):
    """One sequence whose key ``at`` scores ``above`` more than the others' mean, with a value of zero; the others' scores are about
    normal and their values between 1 and 2 (``uneven``: times 2^-5 to 2^5, page by page)."""
    c = Case(kv, qpk, dim, [past], [new], seed=dim + int(above), window=window)
    g = torch.Generator().manual_seed(above)
    k, v = torch.randn(kv, past, dim, generator=g), 1.0 + torch.rand(kv, past, dim, generator=g)
    if uneven:
        v *= 2.0 ** torch.randint(-5, 6, ((past + PAGE - 1) // PAGE,), generator=g).float().repeat_interleave(PAGE)[:past, None]
    k[..., 0] = 0.0
    k[:, at] = 0.0
    k[:, at, 0] = above / (8.0 * c.scale)
    v[:, at] = 0.0
    refill(c, 0, k, v)
    f = c.fused.view(new, kv, qpk + 2, dim)
    f[:, :, :qpk, 0] = 8.0
    f[:, :, qpk, 0] = 0.0
    f[:, :, qpk + 1] = 1.0 + torch.rand(new, kv, dim, generator=g).to(BF)
    return c


def check_positive(c, got, q):
    """All values are positive, so a weight that is off by a part of itself moves the output by no more than that part of it: 2^-11 for a
    float16 number, 2^-12 for scores, exponentials and sums in float32 (scores of some 30 in powers of two, 512 sums of 16 products). Below
    float16's normal numbers a weight is off by half its last place, 2^-25, where the largest is 2^11 or more; the unit of the
    values is at most twice the largest one's: 2^-35 of that a key. The output's own rounding: 2^-8."""
    out, parts = c.attend(q)
    most, keys = parts[0][1], parts[0][3]
    got = got.cpu().double().view(out.shape)
    limit = out * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12) + keys * 2.0 ** -35 * most[..., None]
    assert bool((out > 0).all())
    worst = ((got - out).abs() / out).max()
    assert bool(((got - out).abs() <= limit).all()), f"off by {float(worst):.4f} of the output, allowed {float((limit / out).max()):.4f}"


@pytest.mark.parametrize("above", [8, 14, 16, 18, 20])
@pytest.mark.parametrize("kv,qpk,dim,past", [(2, 4, 128, 8191), (1, 71, 64, 2000), (1, 8, 64, 4000), (1, 12, 128, 3000), (1, 6, 256, 2000), (1, 70, 256, 2000)])
@pytest.mark.parametrize("splits,at,uneven", [(1, 5, False), (1, 1500, True), (2, 0, True), (16, 63, False)])
def test_single_tokens_beside_a_sink(K, kv, qpk, dim, past, above, splits, at, uneven):
    c = beside_a_sink(kv, qpk, dim, past, 1, above, at, uneven)
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, kv, qpk, dim, c.scale, n_splits=splits)
    c.append()
    check_positive(c, out, c.split()[0])
    K.check_device_errors("cuda")


@pytest.mark.parametrize("above", [8, 16, 18, 20])
@pytest.mark.parametrize("kv,qpk,dim,new,tile", [(1, 4, 128, 17, 64), (2, 3, 64, 60, 64), (1, 2, 256, 140, 128), (1, 9, 80, 16, 16)])
@pytest.mark.parametrize("uneven", [False, True])
def test_chunks_beside_a_sink(K, kv, qpk, dim, new, tile, above, uneven):
    c = beside_a_sink(kv, qpk, dim, 2000, new, above, 3, uneven)
    q = c.split()[0].to(BF)
    c.append()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of(c.news, tile)
    out = K.attention_q8(q.cuda(), *cache, batch, *lists, n_tiles, tile, None, kv, c.scale, n_splits=1)
    check_positive(c, out, q.float())
    K.check_device_errors("cuda")


def pages_of_sizes(kv, qpk, dim, sizes, low):
    """A sequence of whole pages whose values are about 2^sizes[i], and a token of its own page in ``low``'s size. Keys of pages of another size
    point away from the queries by hundreds: the weight lies on those of size ``low``."""
    c = Case(kv, qpk, dim, [PAGE * len(sizes)], [1], seed=len(sizes) + dim)
    g = torch.Generator().manual_seed(7)
    n = PAGE * len(sizes)
    k, v = torch.randn(kv, n, dim, generator=g), torch.randn(kv, n, dim, generator=g)
    size = torch.tensor(sizes).repeat_interleave(PAGE)
    v = v.double() * torch.exp2(size.double())[:, None]
    k[..., 0] = torch.where(size == low, 0.0, -50.0 / c.scale)
    refill(c, 0, k, v)
    f = c.fused.view(1, kv, qpk + 2, dim)
    f[:, :, :qpk, 0] = 8.0
    f[:, :, qpk, 0] = 0.0
    f[:, :, qpk + 1] *= 2.0 ** low
    return c, [i for i, e in enumerate(sizes) if e == low]


@pytest.mark.parametrize("kv,qpk,dim", [(1, 1, 64), (2, 3, 128), (1, 20, 128), (1, 71, 64), (1, 9, 256)])
@pytest.mark.parametrize("sizes", [(20, -70), (-70, 20), (20, -120), (-120, 20), (30, -110, 30, -110), (-110, 30, -30, 30, -110, -110), (-126, 60), (60, -126)])
@pytest.mark.parametrize("splits", [1, 2])
def test_small_values_beside_large_ones_without_weight(K, kv, qpk, dim, sizes, splits):
    low = min(sizes)
    c, seen = pages_of_sizes(kv, qpk, dim, sizes, low)
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, kv, qpk, dim, c.scale, n_splits=splits)
    c.append()
    # the other pages' weights are e^-300 and less: the output is that of the seen pages and the new token's
    ids = c.table[0, seen + [len(sizes)]].long()
    k, v = (plain.values(c.codes[x], c.exps[x])[ids].transpose(1, 2).reshape(-1, kv, dim)[:PAGE * len(seen) + 1] for x in "kv")
    want, most, size = plain.attend(c.split()[0], k, v, c.scale, torch.tensor([PAGE * len(seen)]))
    over = (out.cpu().double().view(want.shape) - want).abs() - plain.bound(want, most, size, k.shape[0]) - 2.0 ** -134      # bfloat16's last place
    assert float(most.max()) < 2.0 ** (low + 4) and float(over.max()) <= 0
    K.check_device_errors("cuda")


@pytest.mark.parametrize("kv,qpk,dim", [(1, 2, 64), (2, 1, 128), (1, 2, 256), (1, 5, 80)])
@pytest.mark.parametrize("sizes,window", [((-70, 20), 0), ((-120, 20), 0), ((20, -70, -70), 64), ((20, -120, -120), 64), ((-120, 20, -110, -110), 64)])
@pytest.mark.parametrize("tile", [64, 128])
def test_rows_that_do_not_see_the_large_values(K, kv, qpk, dim, sizes, window, tile):
    # hidden by the causal order, or left of the window: rows of one tile beside others that see them
    n = PAGE * len(sizes)
    c = Case(kv, qpk, dim, [0], [n], window=window, seed=dim)
    f = c.fused.view(n, kv, qpk + 2, dim)
    f[:, :, qpk + 1] *= torch.exp2(torch.tensor(sizes).repeat_interleave(PAGE).float())[:, None, None]
    q = c.split()[0].to(BF)
    c.append()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of(c.news, tile)
    out = K.attention_q8(q.cuda(), *cache, batch, *lists, n_tiles, tile, None, kv, c.scale, window=window)
    c.check(out, q.float())
    K.check_device_errors("cuda")


@pytest.mark.parametrize("e", [-126, -118, -100])
@pytest.mark.parametrize("splits", [1, 3, 16])
def test_the_smallest_values(K, e, splits):
    c = Case(2, 3, 64, [1000], [1], seed=1)
    c.exps["v"][:] = e
    c.fused.view(1, 2, 5, 64)[:, :, 4] *= 2.0 ** e
    cache, batch = c.device(K)
    out = K.attention_decode_q8(c.dev["fused"], *cache, batch, None, None, 2, 3, 64, c.scale, n_splits=splits)
    c.append()
    want, parts = c.attend(c.split()[0])
    over = (out.cpu().double().view(want.shape) - want).abs() - plain.bound(*parts[0]) - 2.0 ** -134
    assert float(over.max()) <= 0 and bool((out != 0).any())


@pytest.mark.parametrize("kv,qpk,dim", [(1, 2, 64), (2, 1, 128), (1, 2, 256), (1, 5, 80)])
@pytest.mark.parametrize("sizes", [(60, -126, -126), (30, 60, -120, -126, -126)])
@pytest.mark.parametrize("tile", [64, 128])
def test_rows_left_of_whose_window_the_largest_values_lie(K, kv, qpk, dim, sizes, tile):
    # up to 2^186 above; the output's own last place is bfloat16's smallest, 2^-133
    n = PAGE * len(sizes)
    c = Case(kv, qpk, dim, [0], [n], window=64, seed=dim)
    f = c.fused.view(n, kv, qpk + 2, dim)
    f[:, :, qpk + 1] *= torch.exp2(torch.tensor(sizes).repeat_interleave(PAGE).float())[:, None, None]
    q = c.split()[0].to(BF)
    c.append()
    cache, batch = c.device(K)
    lists, n_tiles = tiles_of(c.news, tile)
    out = K.attention_q8(q.cuda(), *cache, batch, *lists, n_tiles, tile, None, kv, c.scale, window=64)
    want, parts = c.attend(q.float())
    over = (out.cpu().double().view(want.shape) - want).abs() - plain.bound(*parts[0]) - 2.0 ** -134
    assert float(over.max()) <= 0
    K.check_device_errors("cuda")
