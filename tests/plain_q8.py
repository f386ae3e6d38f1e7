"""The cache in 8 bits in plain form: which codes and exponents appending leaves, what pages stand for, attention over them in 64 bits.

Rounding to e4m3 is written out here (64 bits, nearest, ties to even), apart from any conversion of torch or of the kernels."""
import math

import torch

PAGE = 64
F64 = torch.float64


def exponent(amax: float) -> int:
    """The smallest e in [-126, 119] with amax <= 448 * 2^e."""
    e = -126
    while e < 119 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number of each entry; past 464 (half a step above 448), infinite or no number: no number."""
    y = y.to(F64)
    _, k = torch.frexp(torch.where(torch.isfinite(y), y, torch.zeros_like(y)))
    step = torch.exp2((k - 1).clamp(min=-6).to(F64) - 3)
    r = torch.round(y / step) * step
    return torch.where(y.abs() <= 464.0, r.clamp(-448.0, 448.0), torch.full_like(y, math.nan))


def append(codes, exps, page, first, rows):
    """Rows [kv, n, dim] (float32 or 64) behind the ``first`` rows that the page has; codes [pages, kv, 64, dim] hold e4m3 numbers
    as float64."""
    for g in range(rows.shape[0]):
        x = rows[g].to(F64)
        finite = x[torch.isfinite(x)]
        e = exponent(float(finite.abs().max()) if finite.numel() else 0.0)
        if first > 0:
            old = int(exps[page, g])
            e = max(e, old)
            if e > old:
                codes[page, g, :first] = round_e4m3(codes[page, g, :first] * 2.0 ** (old - e))
        codes[page, g, first:first + x.shape[0]] = round_e4m3(x * 2.0 ** -e)
        exps[page, g] = e


def rotate(x, cos, sin, interleaved):
    """float32 rotation of [tokens, heads, dim], products and sums rounded one by one."""
    if cos is None:
        return x.float()
    n = cos.shape[1]
    x = x.float().clone()
    i = torch.arange(n)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    a, b = x[..., ia].clone(), x[..., ib].clone()
    c, s = cos[:, None], sin[:, None]
    x[..., ia] = a * c - b * s
    x[..., ib] = b * c + a * s
    return x


def values(codes, exps):
    return codes * torch.exp2(exps.to(F64))[..., None, None]


def attend(q, k, v, scale, q_pos, slopes=None, window=0):
    """q [tokens, heads, dim] at positions q_pos over k, v [keys, kv, dim], in 64 bits: outputs [tokens, heads, dim] and, per
    entry, the largest |value| that a row sees and the largest sum of |q k| * scale (for bounds on the error)."""
    heads, kv = q.shape[1], k.shape[1]
    key = torch.arange(k.shape[0])
    seen = key[None, :] <= q_pos[:, None]
    if window:
        seen &= key[None, :] > q_pos[:, None] - window
    out, most, size = torch.zeros(q.shape, dtype=F64), torch.zeros(q.shape[:2], dtype=F64), torch.zeros(q.shape[:2], dtype=F64)
    for h in range(heads):
        g = h // (heads // kv)
        kk, vv = k[:, g].to(F64), v[:, g].to(F64)
        t = q[:, h].to(F64) @ torch.where(seen.any(0)[:, None], kk, torch.zeros((), dtype=F64)).T
        if slopes is not None:
            t = t + (slopes[h].bfloat16() * key.bfloat16()).to(F64)[None]
        p = torch.softmax((t * scale).masked_fill(~seen, -math.inf), -1)
        vv = torch.where(seen.any(0)[:, None], vv, torch.zeros((), dtype=F64))
        out[:, h] = p @ vv
        most[:, h] = torch.stack([vv[s].abs().max() for s in seen])
        big = q[:, h].abs().to(F64) @ kk.abs().T * scale
        size[:, h] = big.masked_fill(~seen, 0).amax(1)
    return out, most, size


def bound(out, most, size, keys, q_bits=11, weight_bits=11):
    """How far a bfloat16 output may be off: rounding the output (2^-8 of it); queries rounded to ``q_bits`` bits (a score moves by at
    most 2^-q_bits * sum |q k| * scale, a normalised weight by twice that in relative terms); weights rounded to ``weight_bits``
    bits, or by half of float16's last place below its normal numbers, 2^-25 a key beside a largest weight of 1 or more; exp2 and sums in float32."""
    score = 2.0 ** -q_bits * size + 1e-5
    weights = torch.expm1(2 * score) + 2.0 ** -weight_bits + keys * 2.0 ** -25 + 1e-5
    return 2.0 ** -8 * out.abs() + (most * weights)[..., None]
