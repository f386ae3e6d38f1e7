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
