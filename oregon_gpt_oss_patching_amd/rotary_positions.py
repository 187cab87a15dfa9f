"""Rotary positions in front of the attention: pairs of a head's numbers turned by their token's angle, with gradients.

    rope = rotary_frequencies(64, 150000.0, factor=32.0, original_length=4096, truncate=False)
    q, k = rotary(q, k, position_ids, rope)            # (B, H, S, D), (B, G, S, D) -> the same shapes
    out = attention(q, k, v, sinks, scale, window, None)

Angles are computed in 64 bits from the positions, so they are as right behind 100000 tokens as in front; the rotation is in 32 bits and
rounded once.  A model that computes its own tables of cosines and sines takes `rotary_tables`, or, patched with
`patch_flash_attention(rotary=True)`, needs nothing else.

The reference leaves the embedding to transformers (its patching.py:6-10 swaps the attention alone).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from . import attention_kernel as _ak

__all__ = ["Rotary", "rotary_frequencies", "rotary", "rotary_tables", "hip_rotary_pos_emb"]


class Rotary(NamedTuple):
    """frequencies: radians of each pair per position, (R / 2) float64 on the GPU (float32 is taken too, a conversion per call); the first R
    numbers of a head are turned, the others go through.  scale: factor of what is turned.  interleaved: numbers 2i and 2i + 1 are pair i, otherwise i and i + R / 2."""
    frequencies: torch.Tensor
    scale: float = 1.0
    interleaved: bool = False


def rotary_frequencies(rotary_dim=64, theta=10000.0, factor=1.0, original_length: Optional[int] = None, beta_fast=32.0, beta_slow=1.0, truncate=True,
                       attention_factor: Optional[float] = None, interleaved=False, device="cuda") -> Rotary:
    """frequencies[i] = theta^(-2i / rotary_dim), for contexts `factor` times as long as those of training:

    * without `original_length`: all divided by `factor` (positions come `factor` times as dense);
    * with it, by parts (the YaRN method): pairs that turn fewer than `beta_slow` times in `original_length` tokens are divided, those that turn more than
      `beta_fast` times kept, those between blended linearly over their number (`truncate`: between whole numbers); the result is scaled by
      `attention_factor`, 0.1 ln(factor) + 1 where none is given."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not theta > 1.0 or not factor > 0.0:
        raise RuntimeError(f"theta must be above 1 and factor positive, got {theta} and {factor}")
    f = theta ** -(torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if original_length is None:
        return Rotary((f / factor).to(device), 1.0 if attention_factor is None else float(attention_factor), bool(interleaved))
    if original_length < 1 or not beta_fast > beta_slow > 0.0:
        raise RuntimeError(f"original_length must be positive and beta_fast > beta_slow > 0, got {original_length}, {beta_fast} and {beta_slow}")

    def pair_of(turns):                          # the (fractional) pair that turns so often in original_length tokens
        return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

    lo, hi = pair_of(beta_fast), pair_of(beta_slow)
    if truncate:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
    divided = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / (hi - lo if hi != lo else 0.001)).clamp(0.0, 1.0)
    if attention_factor is None:
        attention_factor = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return Rotary((f / factor * divided + f * (1.0 - divided)).to(device), float(attention_factor), bool(interleaved))


_ready = False
_op = _now = None           # the operator, and the same without the dispatcher (NotImplemented where it is needed)


def _register_ops() -> None:
    global _ready, _op, _now
    _lib.load_torch_ops()

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::rotary_turn")
    def _turn_fake(q, k, positions, frequencies, cos, sin, scale, interleaved, inverse):
        return tuple(x.new_empty((x.shape[0], x.shape[2], x.shape[1], x.shape[3])).transpose(1, 2) for x in (q, k))

    _now = _lib.direct_calls("gptoss_rotary_direct")
    _op = torch.ops.gptoss_attn.rotary.default
    _ready = True


try:
    _register_ops()
except Exception:       # not built yet: importing has to work for the build itself; the first call tries again and raises
    pass


_compiling = torch.compiler.is_compiling


def _call(q, k, positions, frequencies, cos, sin, scale, interleaved):
    """Through the dispatcher."""
    if positions is not None and not isinstance(positions, torch.Tensor):
        positions = torch.as_tensor(positions, device=q.device)
    return _op(q, k, positions, frequencies, cos, sin, float(scale), bool(interleaved))


def rotary(q, k, positions, rope: Rotary):
    """q (B, H, S, D) and k (B, G, S, D), any strides, D up to 256, turned by their positions' angles: new tensors of the same shapes, whose
    memory is (B, S, heads, D).  `positions`: (B, S), (1, S) or (S) integers, any numbers, negative ones too.

    Differentiable in q and k, any number of times.  float16 goes through float32.  While a graph is recorded with a gradient wanted, q and k must not have eager results
    that are still alive, nor come from an eager call on another stream."""
    if not _ready:
        _register_ops()
    out = NotImplemented if _compiling() else _now(q, k, positions, rope.frequencies, None, None, rope.scale, rope.interleaved)
    return _call(q, k, positions, rope.frequencies, None, None, rope.scale, rope.interleaved) if out is NotImplemented else out


def rotary_tables(q, k, cos, sin, interleaved=False):
    """`rotary` with tables of the angles' cosines and sines, (B, S, R / 2) or (1, S, R / 2), whatever factor they hold."""
    if not _ready:
        _register_ops()
    out = NotImplemented if _compiling() else _now(q, k, None, None, cos, sin, 1.0, interleaved)
    return _call(q, k, None, None, cos, sin, 1.0, interleaved) if out is NotImplemented else out


def hip_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim=1):
    """Drop-in for transformers' `modeling_gpt_oss.apply_rotary_pos_emb`: cos and sin (B, S, D / 2); q and k (B, heads, S, D), or with
    `unsqueeze_dim=2` (B, S, heads, D).  The products are in 32 bits and rounded once, where the eager code rounds each to the model's type.
    Results are of q's and k's type, whatever the tables' (the eager code's are of the wider one: of bfloat16 under autocast with float32 tables, float32)."""
    if unsqueeze_dim == 1:
        return rotary_tables(q, k, cos, sin)
    if unsqueeze_dim != 2:
        raise RuntimeError(f"unsqueeze_dim must be 1, (B, heads, S, D), or 2, (B, S, heads, D), got {unsqueeze_dim}")
    q, k = rotary_tables(q.transpose(1, 2), k.transpose(1, 2), cos, sin)
    return q.transpose(1, 2), k.transpose(1, 2)
