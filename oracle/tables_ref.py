"""Page tables from their definition, a row at a time on the CPU: what gptoss_attn_page_table_update and gptoss_attn_token_map do (the reference has no
counterpart; their definition is that of include/gptoss_attn.h)."""
from __future__ import annotations


def pages_for(n, page_size):
    return -(-max(n, 0) // page_size)


def update(table, have, want, pages, page_size):
    """(table, seqlens, left) of lists; `table` a list of lists."""
    table = [list(row) for row in table]
    width = len(table[0])
    has = [min(pages_for(n, page_size), width) for n in have]
    wants = [pages_for(n, page_size) for n in want]
    kept = [min(h, w) for h, w in zip(has, wants)]
    named = {p for row, k in zip(table, kept) for p in row[:k]}
    free = [p for p in range(pages) if p not in named]
    seqlens, asked, given = [], 0, 0
    for b, row in enumerate(table):
        if wants[b] > width:
            seqlens.append(max(have[b], 0))
            continue
        need = max(0, wants[b] - has[b])
        asked += need
        if need and asked > len(free):
            seqlens.append(max(have[b], 0))
            continue
        row[has[b]:has[b] + need] = free[given:given + need]
        given += need
        for i in range(wants[b], has[b]):
            row[i] = -1
        seqlens.append(max(want[b], 0))
    return table, seqlens, len(free) - given


def token_map(table, start, counts, total, page_size):
    """(row, position, slot, first, used) of lists."""
    row, position, slot, first = [], [], [], []
    for b, n in enumerate(counts):
        begin = len(row)
        for i in range(min(max(n, 0), total - begin)):
            at = start[b] + i
            page = table[b][at // page_size] if 0 <= at < len(table[b]) * page_size else -1
            row.append(b)
            position.append(at)
            first.append(begin)
            slot.append(page * page_size + at % page_size if page >= 0 else -1)
    used = len(row)
    pad = total - used
    return row + [-1] * pad, position + [0] * pad, slot + [-1] * pad, first + [used] * pad, used
