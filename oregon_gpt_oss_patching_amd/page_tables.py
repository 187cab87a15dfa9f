"""Page tables of the cache in pages, built on the GPU from the rows' lengths: who has which page, and where the tokens of a call go.

A scheduler that keeps its lengths on the GPU never has to wait for it: pages are given out, taken back and counted there, and a captured step follows.

    seqlens, left = page_table_update(page_table, have, want, pages, page_size)        # in place; rows grow, shrink, begin and end (want 0)
    tokens = token_map(page_table, have, seqlens - have, total, page_size)             # the call's tokens, back to back
    paged_cache_write_tokens(cache, k, v, tokens.slot)                                 # k, v (total, G, 64)

A page is free iff no row keeps an entry that names it: there is no list of free pages beside the tables, and rows may share pages (a common prefix
copied from one row of the table into another) until the last of them gives them back.  Only full pages: a row's next token goes into its last page where that has room, whoever else
has it.  Where a common prefix ends inside a page, give the new row a page of its own for the rest (an update from the full pages' tokens on) and copy that page's rows in the caches;
and do not let a row that has shrunk into a shared page grow again.  Nothing checks this: such rows overwrite each other's keys and values.

The reference has no counterpart (its generate.py:1-30 leaves the cache to transformers).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from . import attention_kernel as _ak

__all__ = ["TokenMap", "page_table_update", "token_map"]


class TokenMap(NamedTuple):
    """Of each token of a call, back to back in the order of the rows: row (T) int32, position (T) int32 in its row, slot (T) int64 in the pool (-1: none), first (T) int32,
    the number of its row's first token in the call.  Behind the last one: -1, 0, -1 and used.  used (1) int32: how many tokens there are.

    `attention(q, k, v, sinks, scale, window, None, seqlens=used, doc_start=first[None])` is the attention of rows that begin with the call."""
    row: torch.Tensor
    position: torch.Tensor
    slot: torch.Tensor
    first: torch.Tensor
    used: torch.Tensor


_ready = False
_update = _map = None
_update_now = _map_now = None           # the same without the dispatcher, NotImplemented where it is needed


def _register_ops() -> None:
    global _ready, _update, _map, _update_now, _map_now
    _lib.load_torch_ops()

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::page_table_update")
    def _update_fake(page_table, have, want, pages, page_size):
        return page_table.new_empty((page_table.shape[0],)), page_table.new_empty((1,))

    @torch.library.register_fake(f"{_ak.OP_NAMESPACE}::token_map")
    def _map_fake(page_table, start, counts, total, page_size):
        ints = [page_table.new_empty((total,), dtype=torch.int32) for _ in range(3)]
        return ints[0], ints[1], page_table.new_empty((total,), dtype=torch.int64), ints[2], page_table.new_empty((1,), dtype=torch.int32)

    _update_now, _map_now = _lib.direct_calls("gptoss_tables_direct")
    _update, _map = torch.ops.gptoss_attn.page_table_update.default, torch.ops.gptoss_attn.token_map.default
    _ready = True


try:
    _register_ops()
except Exception:       # not built yet: importing has to work for the build itself; the first call tries again and raises
    pass


_compiling = torch.compiler.is_compiling


def _ints(x, like):
    return x if isinstance(x, torch.Tensor) else torch.as_tensor(x, dtype=torch.int32, device=like.device)


def page_table_update(page_table, have, want, pages, page_size):
    """Gives rows of `have` tokens the pages for `want`, in place: page_table (B, width) int32 on the GPU, B up to 16384; have, want (B) integers;
    `pages`: of the pool, up to 2^30.

    A row keeps its first ceil(min(have, want) / page_size) entries and gives the others that it has back (they become -1); free pages go to rows that
    grow in ascending order, row by row.  Where there are too few, the first row that does not get all it wants gets none, nor does any behind it
    that wants some; a row that wants more than its table holds gets none either.  Entries behind a row's pages are left as they are.

    Nothing that runs at the same time may read or write the table; rows of it must not overlap.

    Returns (seqlens (B) int32, left (1) int32): `want` of the rows that have their pages, `have` of the others; the pages that are free now."""
    if not _ready:
        _register_ops()
    out = NotImplemented if _compiling() else _update_now(page_table, have, want, pages, page_size)
    if out is NotImplemented:
        out = _update(page_table, _ints(have, page_table), _ints(want, page_table), int(pages), int(page_size))
    return out


def token_map(page_table, start, counts, total, page_size) -> TokenMap:
    """Where the tokens of a call go that has counts[b] new ones of row b, from position start[b] on, back to back: a `TokenMap` of `total` places,
    which is as many tokens as there may be; those behind it are left out.  B up to 16384."""
    if not _ready:
        _register_ops()
    out = NotImplemented if _compiling() else _map_now(page_table, start, counts, total, page_size)
    if out is NotImplemented:
        out = _map(page_table, _ints(start, page_table), _ints(counts, page_table), int(total), int(page_size))
    return TokenMap(*out)
