"""The key / value cache in pages from its definition, in 64 bits on the CPU: what gptoss_attn_paged_write, _read and _fwd do, a row at a time.

The layer's formula is that of `eager_ref` (the reference's eager attention, attention_kernel.py:36-98); the cache has no counterpart
in the reference (generate.py:1-30 leaves it to transformers), so its definition in include/gptoss_attn.h is what is restated here.
"""
from __future__ import annotations

import torch


def quantise(x):
    """(numbers in units of the row's power of two, exponents) of rows (..., 64): the smallest s >= -64 with the largest finite number at
    most 448 * 2^s, rounded to four significant bits, steps of 2^-9 at least, ties to even; infinities become NaN, and 256 * 2^120, which float32 does not have, 240 * 2^120."""
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    s = torch.full(top.shape, -64, dtype=torch.int64)
    for e in range(-64, 121):
        s = torch.where(top > 448.0 * 2.0 ** e, torch.full_like(s, e + 1), s)
    y = torch.where(finite, x, torch.full_like(x, float("nan"))) / torch.exp2(s.double())
    step = torch.exp2((torch.frexp(y)[1] - 4).clamp(min=-9).double())
    y = torch.round(y / step) * step
    return torch.where((s == 120) & (y.abs() > 240.0), torch.sign(y) * 240.0, y), s[..., 0]


def stored_rows(x, storage):
    """What rows of x stand for once they are in a cache of `storage`."""
    if storage != torch.float8_e4m3fn:
        return x.double()
    y, s = quantise(x)
    return y * torch.exp2(s.double())[..., None]


def page_of(table_row, pos, page_size, pages):
    """Page of a position, None where there is none."""
    if pos < 0 or pos // page_size >= len(table_row):
        return None
    p = int(table_row[pos // page_size])
    return p if 0 <= p < pages else None


def rows_of(pool, table_row, lo, hi, page_size):
    """((G, hi - lo, 64), which of them exist) of positions lo .. hi - 1; pool (pages, G, page_size, 64) in 64 bits."""
    x = torch.zeros(pool.shape[1], max(0, hi - lo), 64, dtype=torch.float64)
    there = torch.zeros(max(0, hi - lo), dtype=torch.bool)
    pos = lo
    while pos < hi:
        n = min(page_size - pos % page_size, hi - pos)
        p = page_of(table_row, pos, page_size, pool.shape[0])
        if p is not None:
            x[:, pos - lo:pos - lo + n] = pool[p, :, pos % page_size:pos % page_size + n]
            there[pos - lo:pos - lo + n] = True
        pos += n
    return x, there


def attention(q, k_pool, v_pool, table, seqlens, sinks, scale, window=0, start=None):
    """(o (B, Sq, H, 64), lse (B, H, Sq), bound terms) in 64 bits; pools hold values.  sinks: (H) or None (a logit of 0).
    The third result is what bounds of a kernel's error are made of: A = sum_j p_j |v_j| like o, the largest scale * sum_d |q_d k_jd| and the
    number of keys of each (B, H, Sq)."""
    b, h, sq, _ = q.shape
    g, ps = k_pool.shape[1], k_pool.shape[2]
    r = h // g
    o = torch.zeros(b, sq, h, 64, dtype=torch.float64)
    amount = torch.zeros_like(o)
    lse = torch.zeros(b, h, sq, dtype=torch.float64)
    size, count = torch.zeros_like(lse), torch.zeros_like(lse)
    sink = (torch.zeros(h) if sinks is None else sinks).double()
    for bi in range(b):
        row = table[bi].tolist()
        n = min(max(int(seqlens[bi]), 0), len(row) * ps)
        for i in range(sq):
            pos = (n - sq if start is None else int(start[bi])) + i
            lse[bi, :, i] = sink
            if pos < 0 or pos >= n:
                continue
            lo = max(0, pos - window + 1) if window else 0
            k, there = rows_of(k_pool, row, lo, pos + 1, ps)
            v, _ = rows_of(v_pool, row, lo, pos + 1, ps)
            if not bool(there.any()):
                continue
            k, v = k[:, there], v[:, there]
            qi = q[bi, :, i].double().view(g, r, 64)
            z = scale * qi @ k.transpose(1, 2)
            sg = sink.view(g, r, 1)
            top = torch.maximum(z.amax(-1, keepdim=True), sg)
            p = torch.exp(z - top)
            total = p.sum(-1, keepdim=True) + torch.exp(sg - top)
            p = p / total
            o[bi, i] = (p @ v).reshape(h, 64)
            amount[bi, i] = (p @ v.abs()).reshape(h, 64)
            lse[bi, :, i] = (top + torch.log(total)).reshape(h)
            size[bi, :, i] = (scale * qi.abs() @ k.abs().transpose(1, 2)).amax(-1).reshape(h)
            count[bi, :, i] = k.shape[1]
    return o, lse, (amount, size, count)


def bounds(o, lse, terms, dtype):
    """How far a kernel's o and lse may be from `attention`'s, element by element.

    With u = 2^-24 (half a step of float32): a logit in 32 bits is a sum of 64 products and up to three scalings, off by at most
    68 u * scale * sum |q k| <= 68 u S; the exponent, taken to base 2, adds the rounding of an argument of at most S + |lse| (times log2 e, back
    times ln 2: (S + |lse|) u, twice, for logit and maximum) and two steps of the exponential itself, 4 u.  So each weight is off
    by at most E = (70 S + 2 |lse| + 4) u of itself, numerator and denominator both: 2 E.  Sums of n such weights and products add n u each.
    For bfloat16 there is room for one rounding of each weight before the second product, half a step of bfloat16: 2^-8 of it (kernels that hold the
    weights in two terms stay far below), and o is rounded once, 2^-8 of o; float32 kernels round o once more, u.  E and n u stay far below 1 in the tests (their second orders: the factor 1.01)."""
    amount, size, count = terms
    u = 2.0 ** -24
    logit = (70 * size + 2 * lse.abs().nan_to_num(posinf=0.0) + 4) * u
    rel = 1.01 * (2 * logit + 2 * (count + 8) * u)
    rel_o = rel.transpose(1, 2)[..., None]
    out = 2.0 ** -8 if dtype == torch.bfloat16 else u
    weight = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    return 1.01 * (rel_o + weight) * amount + out * 1.01 * o.abs() + 1e-37, rel + 4 * u * lse.abs().nan_to_num(posinf=0.0) + 1e-37
