"""A key / value cache in pages and the attention that reads it, for decoding with the layers that `attention` trains.

The sequences of a serving batch share one pool of pages per layer, `PagedCache`, and each has a row of page numbers in a
`page_table` (B, pages of a row): token t stands in slot t % page_size of page page_table[b, t // page_size].  An entry outside
the pool (-1, say) names no page.  The pool holds the model's type, or 8-bit e4m3 numbers with a power of two for each row of
64: half of bfloat16's memory and traffic, each number within 2^-4 of itself; or 4-bit e2m1 numbers with a power of two for each 32 of them: 34 bytes for 128, each
number within a quarter of itself or of that power.

    cache = paged_cache(pages, kv_heads, page_size=64, storage=torch.float8_e4m3fn)      # or torch.float4_e2m1fn_x2
    paged_cache_write(cache, k, v, page_table, start)                     # new tokens' keys and values, (B, G, S, 64)
    out = paged_attention(q, cache, page_table, start + S, sinks, scale, window)      # (B, S, H, 64), as attention()
    k, v = paged_cache_read(cache, page_table, seqlens, max_len)          # rows back, for attention() of a long prompt's chunk

Everything that says where tokens stand (`page_table`, `start`, `seqlens`: integers, numbers beyond int32 being beyond every table) stays on the GPU and
is read there: the calls do not synchronise and can be captured into a graph that is replayed with other contents.  None has a gradient, of either mode.

A patched model takes all of this as one argument, a `PagedState`: `model(ids, position_ids=..., use_cache=False, paged=state)`.

The reference has no counterpart: its generate.py leaves the cache to transformers (generate.py:1-30).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from . import attention_kernel as _ak
from .page_tables import TokenMap

__all__ = ["PagedCache", "PagedState", "paged_cache", "paged_cache_write", "paged_cache_write_tokens", "paged_cache_read", "paged_attention", "paged_attention_forward"]


class PagedCache(NamedTuple):
    """k, v: (pages, G, page_size, 64), bfloat16, float32 or float8_e4m3fn, page_size a power of two from 16 to 1024; rows of 64 must be
    contiguous and start on 16-byte boundaries, the other strides are free.  k_exp, v_exp: float8_e4m3fn only, (pages, G, page_size)
    uint8, a row's values are its numbers times 2^(byte - 127), NaN where the byte is 255.
    float4_e2m1fn_x2: (pages, G, page_size, 32), two numbers to an element, the first in its lower half; exponents (pages, G, page_size, 2), a byte for each half of a row."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: Optional[torch.Tensor] = None
    v_exp: Optional[torch.Tensor] = None


class PagedState(NamedTuple):
    """Where a patched model's layers keep and find their keys and values: `hip_flash_attention(..., paged=PagedState(...))`, which is
    `model(ids, position_ids=..., use_cache=False, paged=PagedState(...))`.

    caches: a `PagedCache` for each layer, by its `layer_idx`.  page_table (B, width): the same pages in each layer's pool.
    start (B): position of each row's first new token; None: the rows begin with this call, and attend to the new tokens as they came.
    seqlens (B): tokens of each row with the new ones.  counts (B): how many of the call's S tokens a row has, where not all have S, the rest being
    padding (start=None: seqlens).  max_len: as in `paged_attention`.
    tokens: a `TokenMap` where the call is one batch row that holds new rows' tokens back to back (start=None, and the map made with starts of 0): the model gets
    tokens.position as its position ids.  (A chunk behind a row's past is a batch row of its own, with start and counts: the attention over pages takes no queries back to back.)"""
    caches: Sequence[PagedCache]
    page_table: torch.Tensor
    start: Optional[torch.Tensor]
    seqlens: torch.Tensor
    counts: Optional[torch.Tensor] = None
    max_len: Optional[int] = None
    tokens: Optional[TokenMap] = None

    def attend(self, module, q, k, v, sm_scale) -> torch.Tensor:
        """A layer's new keys and values into its cache, and its queries' attention."""
        if k.shape[2] != q.shape[2]:
            raise RuntimeError(f"paged= writes the new tokens' keys, as many as queries, got {k.shape[2]} for {q.shape[2]}: the pages hold the past, pass no past_key_values")
        cache, window = self.caches[module.layer_idx], module.sliding_window
        if self.tokens is not None:
            if self.start is not None or q.shape[0] != 1:
                raise RuntimeError(f"tokens= is one batch row of rows that begin with this call: start must be None, got {'one' if self.start is not None else 'none'} and {q.shape[0]} batch rows")
            if self.counts is not None:
                raise RuntimeError("counts= says how many of a batch row's tokens are its own; with tokens= the map says it")
            paged_cache_write_tokens(cache, k[0].transpose(0, 1), v[0].transpose(0, 1), self.tokens.slot)
            return _ak.attention(q, k, v, module.sinks, sm_scale, window, None, self.tokens.used, self.tokens.first[None])
        if self.start is None:
            n = _ints(self.seqlens, q)
            paged_cache_write(cache, k, v, self.page_table, torch.zeros_like(n), n)
            return _ak.attention(q, k, v, module.sinks, sm_scale, window, None, n)
        paged_cache_write(cache, k, v, self.page_table, self.start, self.counts)
        return paged_attention(q, cache, self.page_table, self.seqlens, module.sinks, sm_scale, window, self.start, self.max_len)


def paged_cache(pages, kv_heads, page_size=64, storage=torch.bfloat16, device="cuda") -> PagedCache:
    """An empty cache (all zeros) of one layer."""
    if storage not in (torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float4_e2m1fn_x2):
        raise RuntimeError(f"unsupported storage {storage}: bfloat16, float32, float8_e4m3fn or float4_e2m1fn_x2")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise RuntimeError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
    shape = (pages, kv_heads, page_size)
    if storage == torch.float4_e2m1fn_x2:
        k, v = (torch.zeros((*shape, 32), dtype=torch.uint8, device=device).view(storage) for _ in range(2))
        return PagedCache(k, v, *(torch.zeros((*shape, 2), dtype=torch.uint8, device=device) for _ in range(2)))
    k, v = (torch.zeros((*shape, 64), dtype=storage, device=device) for _ in range(2))
    if storage != torch.float8_e4m3fn:
        return PagedCache(k, v)
    return PagedCache(k, v, *(torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2)))


_ready = False
_write = _read = _fwd = _write_slots = None
_write_now = _read_now = _fwd_now = _write_slots_now = None        # the same without the dispatcher, NotImplemented where it is needed


def _register_ops() -> None:
    global _ready, _write, _read, _fwd, _write_slots, _write_now, _read_now, _fwd_now, _write_slots_now
    _lib.load_torch_ops()
    ops = torch.ops.gptoss_attn

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::paged_write")
    def _write_fake(k_pages, v_pages, k_exp, v_exp, k, v, page_table, start, seqlens):
        return None

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::paged_write_slots")
    def _write_slots_fake(k_pages, v_pages, k_exp, v_exp, k, v, slots):
        return None

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::paged_read")
    def _read_fake(k_pages, v_pages, k_exp, v_exp, page_table, seqlens, max_len, start, dtype):
        shape = (page_table.shape[0], k_pages.shape[1], max_len, 64)
        return k_pages.new_empty(shape, dtype=dtype), k_pages.new_empty(shape, dtype=dtype)

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::paged_fwd")
    def _fwd_fake(q, k_pages, v_pages, k_exp, v_exp, page_table, seqlens, start, sinks, sm_scale, window, max_len, need_lse=True):
        b, h, s, d = q.shape
        return q.new_empty((b, s, h, d)), q.new_empty((b, h, s) if need_lse else (0,), dtype=torch.float32)

    _write_now, _read_now, _fwd_now, _write_slots_now = _lib.direct_calls()
    _write, _read, _fwd, _write_slots = ops.paged_write.default, ops.paged_read.default, ops.paged_fwd.default, ops.paged_write_slots.default
    _ready = True


try:
    _register_ops()
except Exception:       # not built yet: importing has to work for the build itself; the first call tries again and raises
    pass


_Tensor = torch.Tensor
_compiling = torch.compiler.is_compiling


def _ints(x, like):
    return x if x is None or isinstance(x, _Tensor) else torch.as_tensor(x, dtype=torch.int32, device=like.device)


def paged_cache_write(cache: PagedCache, k, v, page_table, start, seqlens=None) -> None:
    """Writes new tokens: k, v (B, G, S, 64), any strides; token i of row b goes to position start[b] + i.  `seqlens`: how many of its S
    tokens each row has, the rest being padding, which is not written.  Positions in front of 0, behind the table, or on an entry that
    names no page are dropped; nothing else of the cache is touched.  float16 tensors are rounded to bfloat16 on the way in, in front of the rounding to codes as well (what is said of a code's
    distance is of the bfloat16 number; a caller who wants float16 numbers rounded once passes them as float32).

    Two rows of one call must not write the same slot, and nothing that runs at the same time may read what is being written."""
    if not _ready:
        _register_ops()
    if _compiling() or _write_now(*cache, k, v, page_table, start, seqlens) is NotImplemented:
        _write(*cache, k, v, _ints(page_table, cache.k), _ints(start, cache.k), _ints(seqlens, cache.k))


def paged_cache_write_tokens(cache: PagedCache, k, v, slots) -> None:
    """`paged_cache_write` of tokens that lie back to back, whatever rows they are of: k, v (T, G, 64), any strides; token t goes to slot
    slots[t], that is to token slots[t] % page_size of page slots[t] // page_size (`token_map` says which).  Slots below 0 or behind the pool are dropped.

    Two tokens of one call must not have the same slot, and nothing that runs at the same time may read what is being written."""
    if not _ready:
        _register_ops()
    if _compiling() or _write_slots_now(*cache, k, v, slots) is NotImplemented:
        slots = slots if isinstance(slots, _Tensor) else torch.as_tensor(slots, dtype=torch.int64, device=cache.k.device)
        _write_slots(*cache, k, v, slots)


def paged_cache_read(cache: PagedCache, page_table, seqlens, max_len, start=None, dtype=None):
    """Rows back out of the pages: k, v (B, G, max_len, 64), row i being position start[b] + i (start: 0).  Zero at and behind seqlens[b], in
    front of 0 and where an entry names no page.  `dtype`: the cache's, or of a cache of codes bfloat16 (exact), float32 or float16.

    The keys and values that a chunk of a long prompt sees, for `attention(q, k, v, sinks, scale, window, start_q)`."""
    if not _ready:
        _register_ops()
    if dtype is None:
        dtype = torch.bfloat16 if cache.k.dtype in (torch.float8_e4m3fn, torch.float4_e2m1fn_x2) else cache.k.dtype
    out = NotImplemented if _compiling() else _read_now(*cache, page_table, seqlens, max_len, start, dtype)
    if out is NotImplemented:
        out = _read(*cache, _ints(page_table, cache.k), _ints(seqlens, cache.k), int(max_len), _ints(start, cache.k), dtype)
    return out


def paged_attention_forward(q, cache: PagedCache, page_table, seqlens, sinks, sm_scale, bandwidth=None, start=None, max_len=None):
    """`paged_attention` that returns (o, lse (B, H, S) float32)."""
    if not _ready:
        _register_ops()
    out = NotImplemented if _compiling() else _fwd_now(q, *cache, page_table, seqlens, start, sinks, sm_scale, bandwidth, max_len, True)
    if out is NotImplemented:
        out = _fwd(q, *cache, _ints(page_table, q), _ints(seqlens, q), _ints(start, q), sinks, float(sm_scale), int(bandwidth or 0), int(max_len or 0))
    return out


def paged_attention(q, cache: PagedCache, page_table, seqlens, sinks, sm_scale, bandwidth=None, start=None, max_len=None):
    """Attention of each row's new queries q (B, H, S, 64) over the row's tokens in the cache, the new ones among them: (B, S, H, 64).

    `seqlens` (B): tokens of each row in the cache.  Query i of row b stands at position start[b] + i (start: seqlens - S, the last S tokens)
    and sees the keys at and before it, with `bandwidth` the last so many of them.  Queries at or behind seqlens[b] are padding: they
    give 0, as does a query that sees no key.  What stands in rows that a query does not see has no part in its result.
    `sinks`, `sm_scale`, `bandwidth`: as in `attention` (sinks=None: a logit of 0; logits of -inf: no sink).
    `max_len`: a length that no row passes, if the caller knows one shorter than the table; it only helps to divide the work: rows that are known to be short (up
    to some 1000 to 3000 tokens, by their type and number) take one launch and not two.

    The cache is read once for each 64 pairs of a query and a head of its KV head's group (32 in float32); the many queries of a prompt's chunk are
    better served by `paged_cache_read` and `attention`."""
    if not _ready:
        _register_ops()
    out = NotImplemented if _compiling() else _fwd_now(q, *cache, page_table, seqlens, start, sinks, sm_scale, bandwidth, max_len, False)
    if out is NotImplemented:
        out = _fwd(q, *cache, _ints(page_table, q), _ints(seqlens, q), _ints(start, q), sinks, float(sm_scale), int(bandwidth or 0), int(max_len or 0),
                   False)[0]
    return out
