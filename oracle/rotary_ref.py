"""Rotary positions from their definition, in 64 bits on the CPU: pairs of numbers as complex ones, multiplied by scale * exp(i p f).

What the model's own embedding computes in its type (transformers' apply_rotary_pos_emb, in front of the reference's attention).
"""
from __future__ import annotations

import torch


def pairs_of(x, turned, interleaved):
    """The first `turned` numbers of each row (..., D) as (..., turned / 2) complex numbers."""
    part = x[..., :turned].double()
    part = part.unflatten(-1, (-1, 2)) if interleaved else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    return torch.complex(part[..., 0], part[..., 1])


def turn(x, z, interleaved=False):
    """x (B, heads, S, D), z complex (B or 1, S, pairs): each pair times its z, in 64 bits."""
    turned = 2 * z.shape[-1]
    y = torch.view_as_real(pairs_of(x, turned, interleaved) * z[:, None])
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., turned:].double()), -1)


def of_positions(positions, frequencies, scale=1.0):
    """z of positions (B, S) and frequencies in 64 bits."""
    angle = positions.double()[..., None] * frequencies.double()
    return torch.polar(torch.full_like(angle, scale), angle)


def of_tables(cos, sin):
    return torch.complex(cos.double(), sin.double())


def bound(x, z, y, dtype, interleaved=False, angles=True):
    """How far a kernel's result may be from y = turn(x, z), element by element.

    With u = 2^-24 (half a step of float32), for a pair of magnitudes a1, a2 under a factor of magnitude m = |z|: cosine and sine are off by at most 4 u before the
    scale (of tables: nothing), whose own rounding and the product's add 2 u, so each is off by 6 u m; an angle in 64 bits that is off by 2^-30 at most (positions
    below 2^21) adds 2^-6 u m.  The two products and their sum round twice more, 2 u m (a1 + a2).  So 8.1 u m (a1 + a2), and the result's own rounding:
    2^-8 of it in bfloat16, in float32 that of the sum, counted already."""
    u = 2.0 ** -24
    turned = 2 * z.shape[-1]
    p = pairs_of(x, turned, interleaved)
    amount = (p.real.abs() + p.imag.abs()) * z.abs()[:, None] * (8.1 if angles else 2.1) * u
    amount = amount.repeat_interleave(2, -1) if interleaved else torch.cat((amount, amount), -1)
    amount = torch.cat((amount, torch.zeros_like(y[..., turned:])), -1)
    if dtype == torch.bfloat16:
        amount[..., :turned] += 2.0 ** -8 * 1.01 * y[..., :turned].abs()
    return amount + 1e-40
