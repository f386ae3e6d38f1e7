"""Cases that stand for what programs do with a paged cache of keys and values held in 8 bits: append to it, attend over
it, and copy its pages. Each is computed in a plain form of elementary torch operations, or by the library's kernels.

The cache. A page holds 64 tokens of one key/value head as e4m3 codes ``[pages, kv_heads, 64, dim]`` and one exponent
``[pages, kv_heads]``: a value is code * 2^exponent. Appending rows to a page:

* the exponent that rows need is the smallest e in [-126, 119] with max |x| <= 448 * 2^e over their finite entries;
* a page that gets its first token takes what the new rows need; a page with earlier tokens takes the larger of that and
  its own, and if its own rose, the earlier codes are rounded again: e4m3(code * 2^(old - new));
* new codes are e4m3(x * 2^-e), rounded to nearest even; what is infinite or no number is held as no number;
* rows behind the last token keep their codes.

Kinds of cases:

* ``decode``   one new token for each sequence: queries and key rotated, key and value appended, attention over the cache.
               Outputs: the attention's rows, and the values of the pages that the step wrote to.
* ``store``    a step's projection into rotated queries and appended keys and values, as prompts do it. Outputs: the
               queries, and the values of the pages that the step wrote to.
* ``prompt``   attention of many new tokens a sequence over pages that hold them and their past already.
* ``copy``     pages of several tensors of pages copied, within them or into others. Outputs: the tensors.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 64
F8 = torch.float8_e4m3fn
F64 = torch.float64
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one chat on Falcon-7B (71 heads on one key/value head): a step's smallest attention, where latency counts
        dict(name="decode 7b one", kind="decode", seqs=1, context=2047, ragged=0.0, kv=1, qpk=71, dim=64, position="half", rot=64,
             window=0),
        # eight chats of very different lengths on Falcon-11B (32 heads on 8, heads of 128)
        dict(name="decode 11b ragged", kind="decode", seqs=8, context=4095, ragged=1.0, kv=8, qpk=4, dim=128, position="half",
             rot=128, window=0),
        # one long document on Falcon-40B (128 heads on 8): few rows, so the keys are split over the device
        dict(name="decode 40b long", kind="decode", seqs=1, context=32767, ragged=0.0, kv=8, qpk=16, dim=64, position="half",
             rot=64, window=0),
        # a full serving batch at long contexts, Falcon-11B: what the cache's bytes bind
        dict(name="decode 11b batch", kind="decode", seqs=64, context=8191, ragged=0.3, kv=8, qpk=4, dim=128, position="half",
             rot=128, window=0),
        # heads of 80, three to a group, ALiBi, a sliding window that ends inside a page
        dict(name="decode window alibi", kind="decode", seqs=5, context=3001, ragged=0.5, kv=2, qpk=3, dim=80, position="alibi",
             rot=0, window=1000),
        # three prompts of odd lengths on Falcon-11B, the second after 70 tokens of its own
        dict(name="store prompts", kind="store", seqs=3, new=967, ragged=0.4, past=70, kv=8, qpk=4, dim=128, position="half", rot=128),
        # 64 single tokens on Falcon-40B, half of a head rotated in adjacent pairs: pages whose exponent may rise
        dict(name="store tokens", kind="store", seqs=64, new=1, ragged=0.0, past=1000, kv=8, qpk=16, dim=64, position="pairs", rot=32),
        # short continuations (a turn of a conversation, a checked draft) after long pasts, Falcon-11B
        dict(name="prompt short chunks", kind="prompt", seqs=4, new=17, ragged=0.5, past=3000, kv=8, qpk=4, dim=128,
             position="none", window=0),
        # a whole prompt on Falcon-11B: bound by the matrix products
        dict(name="prompt 11b", kind="prompt", seqs=1, new=3500, ragged=0.0, past=0, kv=8, qpk=4, dim=128, position="none", window=0),
        # two chunks of prompts with heads of 96, ALiBi and a window
        dict(name="prompt odd heads", kind="prompt", seqs=2, new=777, ragged=0.3, past=500, kv=3, qpk=2, dim=96, position="alibi",
             window=600),
        # a sequence of Falcon-11B forked into four: the last, partly filled page of 60 layers' keys and values
        dict(name="copy fork", kind="copy", entries=60, pages=200, kv=8, dim=128, dtype="float8_e4m3fn", pairs=4, mode="fork"),
        # a bfloat16 cache moved into a larger one: 400 pages of 32 layers, Falcon-7B
        dict(name="copy resize", kind="copy", entries=32, pages=600, kv=1, dim=64, dtype="bfloat16", pairs=400, mode="other"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


#: What no drawn case costs more than: bytes of keys and values, operations on prompts, bytes copied
_MOST_CACHE = 64 * 8191 * 8 * 128 * 2 * 0.8
_MOST_FLOPS = 1e11
_MOST_COPIED = 32 * 400 * 64 * 64 * 2 * 2


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "store", "prompt", "prompt", "copy"])
    dim = rng.choice([64, 64, 128, 128, 16, 32, 48, 80, 96, 112, 192, 256])
    kv = rng.choice([1, 1, 2, 3, 4, 8, 8])
    qpk = min(_log(rng, 1, 71), 128 // kv if kind == "prompt" else 71)
    position = rng.choice(["half", "half", "pairs", "alibi", "none"])
    rot = 0 if position in ("alibi", "none") else rng.choice([dim, dim // 2])
    c = dict(kind=kind, kv=kv, qpk=qpk, dim=dim, position=position, rot=rot)
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        context = int(min(_log(rng, 1, 40000) - 1, _MOST_CACHE / (seqs * kv * dim * 2)))
        window = rng.choice([0, 0, 0, 1, 63, 64, _log(rng, 2, 5000)])
        return dict(c, seqs=seqs, context=context, ragged=rng.choice([0.0, 0.5, 1.0]), window=window)
    if kind == "store":
        seqs = _log(rng, 1, 48)
        new = rng.choice([1, _log(rng, 2, max(3, 3000 // seqs))])
        return dict(c, seqs=seqs, new=new, ragged=rng.choice([0.0, 0.6]), past=rng.choice([0, _log(rng, 1, 2000)]))
    if kind == "prompt":
        c.pop("rot")
        c["position"] = rng.choice(["none", "none", "alibi"])
        seqs = rng.choice([1, 1, 2, 3])
        past = rng.choice([0, 0, _log(rng, 1, 4000)])
        new = _log(rng, 2, 3000)
        while 4 * kv * qpk * dim * seqs * (new * past + new * (new + 1) / 2) > _MOST_FLOPS:
            new, past = max(2, new * 3 // 4), past * 3 // 4
        return dict(c, seqs=seqs, new=new, ragged=rng.choice([0.0, 0.5]), past=past,
                    window=rng.choice([0, 0, 0, _log(rng, 1, 2000)]))
    dtype = rng.choice(["float8_e4m3fn", "bfloat16", "float32"])
    entries = _log(rng, 1, 60)
    size = {"float8_e4m3fn": 1, "bfloat16": 2, "float32": 4}[dtype]
    pairs = max(1, min(_log(rng, 1, 1500), int(_MOST_COPIED / (entries * kv * PAGE * dim * size * 2))))
    return dict(kind=kind, entries=entries, pages=2 * pairs + rng.randrange(1, 40), kv=kv, dim=dim, dtype=dtype, pairs=pairs,
                mode=rng.choice(["fork", "move", "other"]))


# ------------------------------------------------------------------------------------------------ sizes of a case
def _spread(most, ragged, seqs, low):
    """Lengths from ``most`` down by up to the share ``ragged``, in no order; they follow from the case alone."""
    return [max(low, most - int(most * ragged * ((7 * i + 3) * i % 11) / 11)) for i in range(seqs)]


def _lengths(c):
    """(past, new) tokens of each sequence."""
    if c["kind"] == "decode":
        return [(p, 1) for p in _spread(c["context"], c["ragged"], c["seqs"], 0)]
    new = _spread(c["new"], c["ragged"], c["seqs"], 1)
    # every third sequence has no past
    return [(c["past"] if i % 3 == 1 or c["past"] == 0 or c["kind"] == "prompt" or c["new"] == 1 else 0, n) for i, n in enumerate(new)]


def _visible(p, n, window):
    """(keys that some query of the sequence sees, pairs of a query and a key that it sees)."""
    total = p + n
    if not window:
        return total, n * p + n * (n + 1) // 2
    return min(total, n + window - 1), sum(min(q + 1, window) for q in range(p, total))


def _touched(c):
    """Pages that the new tokens lie in."""
    return sum((p + n - 1) // PAGE - p // PAGE + 1 for p, n in _lengths(c))


def work(case):
    c = case
    if c["kind"] == "copy":
        size = {"float8_e4m3fn": 1, "bfloat16": 2, "float32": 4}[c["dtype"]]
        page = c["entries"] * 2 * c["kv"] * (PAGE * c["dim"] * size + (1 if size == 1 else 0))
        sources = c["pairs"] if c["mode"] != "fork" else (c["pairs"] + 3) // 4
        return {"bytes": page * (sources + c["pairs"]), "flops": 0}
    lengths = _lengths(c)
    kv, dim, heads = c["kv"], c["dim"], c["kv"] * c["qpk"]
    tokens = sum(n for _, n in lengths)
    width = kv * (c["qpk"] + 2) * dim
    seen = [_visible(p, n, c.get("window", 0)) for p, n in lengths]
    rows = 2 * kv * dim                              # a token's codes, keys and values
    read_back = _touched(c) * kv * PAGE * dim * 2 * (1 + 2)      # the written pages' codes, and their values in 16 bits
    if c["kind"] == "store":
        return {"bytes": tokens * (width + heads * dim) * 2 + tokens * rows + tokens * c["rot"] * 4 + read_back, "flops": 0}
    flops = 4 * heads * dim * sum(pairs for _, pairs in seen)
    keys = sum(k for k, _ in seen) * rows
    if c["kind"] == "decode":
        return {"bytes": keys + tokens * (width + heads * dim) * 2 + tokens * rows + tokens * c["rot"] * 4 + read_back, "flops": flops}
    return {"bytes": keys + 2 * tokens * heads * dim * 2, "flops": flops}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _power(e):
    """2^e in float32, exactly (e a tensor of whole numbers in [-126, 127])."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _needed(amax):
    """The smallest e in [-126, 119] with amax <= 448 * 2^e."""
    m, k = torch.frexp(amax)          # amax = m 2^k, m in [0.5, 1); 448 = 0.875 * 2^9
    e = k - 9 + (m > 0.875).to(k.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(-126, 119)


def _pool(gen, pages, kv, dim, spread):
    """Pages as tokens before have left them: normal entries, heads of different sizes, a few outlying entries."""
    head = 2.0 ** (spread * torch.randn(kv, generator=gen, device=DEV))
    x = torch.randn(pages, kv, PAGE, dim, generator=gen, device=DEV) * head[None, :, None, None]
    x[:, :, :, 0] *= 6.0
    e = _needed(x.abs().amax((2, 3)))
    return (x * _power(-e)[..., None, None]).to(F8), e.to(torch.int8)


def _tiles(lengths):
    """(sequence, first new token) every 16, 64 or 128 tokens by the longest sequence, longest walks first."""
    longest = max(n for _, n in lengths)
    size = 16 if longest <= 16 else 64 if longest <= 64 else 128
    tiles = [(b, q0) for b, (_, n) in enumerate(lengths) for q0 in range(0, n, size)]
    tiles.sort(key=lambda t: -(lengths[t[0]][0] + t[1]))
    return size, [b for b, _ in tiles], [q for _, q in tiles]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if c["kind"] == "copy":
        shape = (c["entries"], c["pages"], c["kv"], PAGE, c["dim"])
        dtype = getattr(torch, c["dtype"])
        if dtype == F8:
            pools = [torch.randint(0, 127, shape, generator=gen, device=DEV, dtype=torch.uint8).view(F8) for _ in range(2)]
            pools += [torch.randint(-9, 9, shape[:3], generator=gen, device=DEV, dtype=torch.int8) for _ in range(2)]
        else:
            pools = [torch.randn(shape, generator=gen, device=DEV).to(dtype) for _ in range(2)]
        order = np.random.RandomState(seed % (1 << 31)).permutation(c["pages"]).astype(np.int32)
        n = c["pairs"]
        src, dst = order[:n], order[n:2 * n]
        if c["mode"] == "fork":          # every source for four sequences
            src = np.repeat(src, 4)[:n].copy()
        others = None
        if c["mode"] == "other":         # into the low pages of other storage
            others = [torch.zeros_like(p) for p in pools]
            dst = np.arange(n, dtype=np.int32)
        return dict(kind="copy", pools=pools, others=others, src=src, dst=dst, src_dev=torch.from_numpy(src).long().to(DEV),
                    dst_dev=torch.from_numpy(dst).long().to(DEV))
    lengths = _lengths(c)
    seqs, kv, qpk, dim = len(lengths), c["kv"], c["qpk"], c["dim"]
    heads, tokens = kv * qpk, sum(n for _, n in lengths)
    counts = [(p + n + PAGE - 1) // PAGE for p, n in lengths]
    pool_pages = sum(counts) + 3
    k_pool, k_exp = _pool(gen, pool_pages, kv, dim, 0.5)
    v_pool, v_exp = _pool(gen, pool_pages, kv, dim, 1.0)
    order = random.Random(seed).sample(range(pool_pages), pool_pages)
    table = np.full((seqs, max(counts)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
        if c.get("window", 0):           # pages that no query of the step sees have been given back
            table[b, :max(0, lengths[b][0] - c["window"] + 1) // PAGE] = -1
    start = np.cumsum([0] + [n for _, n in lengths])
    seq_of = np.repeat(np.arange(seqs), [n for _, n in lengths])
    pos = np.concatenate([np.arange(p, p + n) for p, n in lengths])
    # the pages that the step writes to: (sequence, page of the sequence)
    written = [(b, i) for b, (p, n) in enumerate(lengths) for i in range(p // PAGE, (p + n - 1) // PAGE + 1)]

    def ints(x):
        return torch.as_tensor(np.asarray(x, dtype=np.int32), device=DEV).contiguous()

    s = dict(kind=c["kind"], kv=kv, qpk=qpk, dim=dim, window=c.get("window", 0), scale=1.0 / math.sqrt(dim), k_pool=k_pool,
             k_exp=k_exp, v_pool=v_pool, v_exp=v_exp, table=ints(table), tok_seq=ints(seq_of), tok_pos=ints(pos),
             seq_start=ints(start[:-1]), seq_new=ints([n for _, n in lengths]), seq_past=ints([p for p, _ in lengths]),
             pages=sum(counts), interleaved=c["position"] == "pairs", rope=None, slopes=None)
    if c["position"] == "alibi":
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV) / heads)).bfloat16().float()
    if c["kind"] == "prompt":
        s["tile_tokens"], tile_seq, tile_q0 = _tiles(lengths)
        s["tile_seq"], s["tile_q0"] = ints(tile_seq), ints(tile_q0)
        s["q"] = torch.randn(tokens, heads, dim, generator=gen, device=DEV).mul_(1.2).bfloat16()
        s["most_new"], s["most"] = max(n for _, n in lengths), max(counts)
        return s
    if c["rot"]:
        freq = 1.0 / (10000.0 ** (torch.arange(0, c["rot"], 2, device=DEV, dtype=F64) / c["rot"]))
        angle = s["tok_pos"].to(F64)[:, None] * freq[None, :]
        s["rope"] = (angle.cos().float(), angle.sin().float())
    fused = torch.randn(tokens, kv, qpk + 2, dim, generator=gen, device=DEV)
    fused[:, :, qpk:] *= 2.0 ** torch.randn(tokens, kv, 1, 1, generator=gen, device=DEV)    # now and then an exponent rises
    s["fused"] = fused.bfloat16().reshape(tokens, kv * (qpk + 2) * dim)
    s["written_seq"], s["written_page"] = ints([b for b, _ in written]).long(), ints([i for _, i in written]).long()
    s["written"] = ints([table[b, i] for b, i in written])
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _values(pool, exps, ids):
    return pool[ids].float() * _power(exps[ids])[..., None, None]


def _rotate(x, rope, interleaved):
    """``x`` [tokens, heads, dim] float32, its first 2 * pairs entries rotated in pairs (i, i + pairs) or (2 i, 2 i + 1)."""
    if rope is None:
        return x
    cos, sin = rope[0][:, None], rope[1][:, None]
    n = cos.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _append(s, pool, exps, rows):
    """``rows`` [tokens, kv, dim] float32 into the written pages."""
    ids, seq = s["written"].long(), s["written_seq"]
    slot = torch.arange(PAGE, device=DEV)
    pos = s["written_page"][:, None] * PAGE + slot                        # [written, 64]
    past, start = s["seq_past"].long()[seq][:, None], s["seq_start"].long()[seq][:, None]
    fresh = (pos >= past) & (pos < past + s["seq_new"].long()[seq][:, None])
    earlier = pos < past
    x = rows[(start + pos - past).clamp(0, rows.shape[0] - 1)].transpose(1, 2)      # [written, kv, 64, dim]
    use = fresh[:, None, :, None]
    x = torch.where(torch.isfinite(x), x, torch.full_like(x, math.nan))
    need = _needed(torch.where(use & torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((2, 3)))
    old = exps[ids].to(need.dtype)
    e = torch.where(earlier[:, :1], torch.maximum(old, need), need)
    had = pool[ids].float()
    again = had * torch.exp2((old - e).clamp(-140, 0).double()).float()[..., None, None]
    codes = torch.where(use, x * _power(-e)[..., None, None], torch.where(earlier[:, None, :, None], again, had))
    pool[ids] = codes.to(F8)
    exps[ids] = e.to(torch.int8)


def _split(s):
    """Rotated queries and keys, and values, in float32."""
    f = s["fused"].float().view(-1, s["kv"], s["qpk"] + 2, s["dim"])
    tokens = f.shape[0]
    q = _rotate(f[:, :, :s["qpk"]].reshape(tokens, -1, s["dim"]), s["rope"], s["interleaved"])
    return q, _rotate(f[:, :, s["qpk"]], s["rope"], s["interleaved"]), f[:, :, s["qpk"] + 1]


def _attend(s, q, q_pos):
    """``q`` [seqs, kv, qpk, tokens, dim] float32 at positions ``q_pos`` [seqs, tokens] (-1: no token): attention over the pages."""
    seqs, kv, qpk, n, dim = q.shape
    ids = s["table"].long().clamp(min=0)

    def rows(pool, exps):
        return _values(pool, exps, ids).transpose(1, 2).reshape(seqs, kv, -1, dim)

    k = rows(s["k_pool"], s["k_exp"])
    scores = (q.reshape(seqs, kv, qpk * n, dim) @ k.transpose(2, 3)).view(seqs, kv, qpk, n, -1)
    key = torch.arange(k.shape[2], device=DEV)
    if s["slopes"] is not None:
        bias = (s["slopes"].bfloat16()[:, None] * key.bfloat16()[None, :]).float()          # rounded as the framework rounds it
        scores = scores + bias.view(1, kv, qpk, 1, -1)
    seen = key <= q_pos[:, :, None]
    if s["window"]:
        seen = seen & (key > q_pos[:, :, None] - s["window"])
    scores = (scores * s["scale"]).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    # a given-back page's table entry is -1: nothing of it counts, whatever the page in its place holds
    v = torch.where(seen.any(1)[:, None, :, None], rows(s["v_pool"], s["v_exp"]), torch.zeros((), device=DEV))
    return (p.view(seqs, kv, qpk * n, -1) @ v).view(seqs, kv, qpk, n, dim) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain(s):
    if s["kind"] == "copy":
        into = s["others"] or s["pools"]
        return [_copied(p, o, s) for p, o in zip(s["pools"], into)]
    if s["kind"] == "prompt":
        seqs, most = s["seq_new"].numel(), s["most_new"]
        i = torch.arange(most, device=DEV)[None, :]
        new = s["seq_new"].long()[:, None]
        at = (s["seq_start"].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)
        pos = torch.where(i < new, s["seq_past"].long()[:, None] + i, torch.full_like(at, -1))
        q = s["q"].float()[at].view(seqs, most, s["kv"], s["qpk"], s["dim"]).permute(0, 2, 3, 1, 4)
        o = _attend(s, q, pos).permute(0, 3, 1, 2, 4).reshape(seqs, most, -1)
        return o[i < new].bfloat16()
    q, k, v = _split(s)
    _append(s, s["k_pool"], s["k_exp"], k)
    _append(s, s["v_pool"], s["v_exp"], v)
    ids = s["written"].long()
    pages = [_values(s["k_pool"], s["k_exp"], ids).bfloat16(), _values(s["v_pool"], s["v_exp"], ids).bfloat16()]
    if s["kind"] == "store":
        return [q.bfloat16()] + pages
    o = _attend(s, q.view(-1, s["kv"], s["qpk"], 1, s["dim"]), s["seq_past"].long()[:, None])
    return [o.reshape(q.shape[0], -1).bfloat16()] + pages


def _copied(pool, into, s):
    # pages are copied as bytes: what 8 bits stand for does not matter to it, and numbers that are no number stay as they are
    a, b = (pool.view(torch.uint8), into.view(torch.uint8)) if pool.element_size() == 1 else (pool, into)
    b[:, s["dst_dev"]] = a[:, s["src_dev"]]
    return b


# ------------------------------------------------------------------------------------------------ the library's kernels
def _kernels(s):
    from pytorch_transformers_b200 import kernels as K
    if s["kind"] == "copy":
        into = K.copy_pages(s["pools"], s["src"], s["dst"], out=s["others"])
        return [p.view(torch.uint8) if p.element_size() == 1 else p for p in into]
    batch = K.step_batch(s["tok_seq"], s["tok_pos"], s["seq_start"], s["seq_new"], s["seq_past"], s["table"])
    cache = (s["k_pool"], s["k_exp"], s["v_pool"], s["v_exp"])
    if s["kind"] == "prompt":
        return K.attention_q8(s["q"], *cache, batch, s["tile_seq"], s["tile_q0"], s["tile_seq"].numel(), s["tile_tokens"], s["slopes"],
                              s["kv"], s["scale"], window=s["window"], n_pages=s["pages"])
    if s["kind"] == "store":
        out = K.split_rotate_store_q8(s["fused"], *cache, batch, s["kv"], s["qpk"], s["dim"], rope=s["rope"],
                                      interleaved=s["interleaved"])
    else:
        out = K.attention_decode_q8(s["fused"], *cache, batch, s["rope"], s["slopes"], s["kv"], s["qpk"], s["dim"], s["scale"],
                                    window=s["window"], interleaved=s["interleaved"])
    return [out, *K.unpack_pages_q8(*cache, s["written"])]


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _round_e4m3(y):
    """The nearest e4m3 number of y (64 bits, |y| <= 448), ties to even."""
    _, k = torch.frexp(y)
    step = torch.exp2((k - 1).clamp(min=-6).to(F64) - 3)
    return torch.round(y / step) * step


def _exact_append(s, pool, exps, rows):
    """Values [pages, kv, 64, dim] in 64 bits after the step, sequence by sequence, page by page."""
    scale = torch.exp2(exps.to(F64))
    codes = {}
    for b in range(s["seq_new"].numel()):
        past, new, start = (int(s[n][b]) for n in ("seq_past", "seq_new", "seq_start"))
        for i in range(past // PAGE, (past + new - 1) // PAGE + 1):
            page = int(s["table"][b, i])
            lo, hi = max(past, i * PAGE), min(past + new, (i + 1) * PAGE)
            x = rows[start + lo - past:start + hi - past].transpose(0, 1)         # [kv, tokens, dim]
            amax = x.abs().amax((1, 2))
            e = torch.ceil(torch.log2(amax / E4M3_MAX).clamp(-126, 119))
            e = torch.where(amax <= E4M3_MAX * torch.exp2(e - 1), e - 1, torch.where(amax > E4M3_MAX * torch.exp2(e), e + 1, e)).clamp(-126, 119)
            old = exps[page].to(F64)
            if lo > i * PAGE:
                e = torch.maximum(e, old)
            code = pool[page].to(F64)
            first, last = lo - i * PAGE, hi - i * PAGE
            code[:, :first] = _round_e4m3(code[:, :first] * torch.exp2(old - e)[:, None, None])
            code[:, first:last] = _round_e4m3(x * torch.exp2(-e)[:, None, None])
            scale[page] = torch.exp2(e)
            codes[page] = code
    return codes, scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        if case["dtype"] == "float8_e4m3fn":
            return None          # bytes: whole numbers, equal or wrong
        before, after = [[p.to(F64) for p in (pools or [])] for pools in (s["pools"], s["others"])]
        after = after or [p.clone() for p in before]
        for a, b in zip(before, after):
            for src, dst in zip(s["src"].tolist(), s["dst"].tolist()):
                b[:, dst] = a[:, src]
        return after
    kv, qpk, dim, scale = s["kv"], s["qpk"], s["dim"], s["scale"]
    pages = []
    changed = {"k_pool": ({}, torch.exp2(s["k_exp"].to(F64))), "v_pool": ({}, torch.exp2(s["v_exp"].to(F64)))}
    if case["kind"] == "prompt":
        q = s["q"].to(F64)
    else:
        f = s["fused"].to(F64).view(-1, kv, qpk + 2, dim)
        q, k, v = f[:, :, :qpk].reshape(-1, kv * qpk, dim).clone(), f[:, :, qpk].clone(), f[:, :, qpk + 1].clone()
        if s["rope"] is not None:
            n = s["rope"][0].shape[1]
            one = torch.arange(n, device=DEV)
            first, second = (2 * one, 2 * one + 1) if s["interleaved"] else (one, one + n)
            c, d = s["rope"][0].to(F64)[:, None], s["rope"][1].to(F64)[:, None]
            for x in (q, k):
                a, b = x[..., first], x[..., second]
                x[..., first], x[..., second] = a * c - b * d, a * d + b * c
        for name, rows in (("k", k), ("v", v)):
            codes, factor = changed[name + "_pool"] = _exact_append(s, s[name + "_pool"], s[name + "_exp"], rows)
            pages.append(torch.stack([codes[p] * factor[p][:, None, None] for p in s["written"].tolist()]))
        if case["kind"] == "store":
            return [q] + pages
    out = torch.zeros(q.shape[0], kv * qpk, dim, dtype=F64, device=DEV)
    for b in range(s["seq_new"].numel()):
        past, new, start = (int(s[n][b]) for n in ("seq_past", "seq_new", "seq_start"))
        low = max(0, past - s["window"] + 1) // PAGE if s["window"] else 0
        ids = s["table"][b, low:(past + new + PAGE - 1) // PAGE].tolist()

        def of(name):
            codes, factor = changed[name]
            at = torch.tensor(ids, device=DEV)
            values = s[name][at].to(F64)
            for i, p in enumerate(ids):
                if p in codes:
                    values[i] = codes[p]
            return (values * factor[at][..., None, None]).transpose(0, 1).reshape(kv, -1, dim)[:, :past + new - low * PAGE]

        keys, values = of("k_pool"), of("v_pool")
        key = torch.arange(low * PAGE, past + new, device=DEV)
        pos = torch.arange(past, past + new, device=DEV)[:, None]
        hidden = key[None] > pos
        if s["window"]:
            hidden |= key[None] <= pos - s["window"]
        for h in range(kv * qpk):
            t = q[start:start + new, h] @ keys[h // qpk].T
            if s["slopes"] is not None:
                t = t + (s["slopes"][h].bfloat16() * key.bfloat16()).to(F64)
            out[start:start + new, h] = torch.softmax((t * scale).masked_fill(hidden, -math.inf), -1) @ values[h // qpk]
    out = out.reshape(q.shape[0], -1)
    return out if case["kind"] == "prompt" else [out] + pages
