"""A pool of cache pages in plain Python, request by request: what
paged_cache_extend and paged_cache_release do."""
from __future__ import annotations


def extend(table, lengths, counts, pool, page, tokens):
    """Changes `table` (lists of pages) and `pool` (a list, its end the top) in place.
    Returns (slots, positions, cu_seqlens, lengths) of the granted tokens."""
    slots, positions, cu, after = [], [], [0], []
    asked, wanted, free = 0, 0, len(pool)
    for row, length, count in zip(table, lengths, counts):
        count = max(count, 0)
        asked += count
        granted = length >= 0 and asked <= tokens and length + count <= len(row) * page
        if granted:
            held, rows = -(-length // page), -(-(length + count) // page)
            wanted += rows - held
            granted = rows == held or wanted <= free
        if granted:
            for i in range(held, rows):
                row[i] = pool.pop()
            for p in range(length, length + count):
                slots.append(row[p // page] * page + p % page if row[p // page] >= 0 else -1)
                positions.append(p)
        after.append(length + count if granted else length)
        cu.append(len(slots))
    pad = [-1] * (tokens - len(slots))
    return slots + pad, positions + pad, cu, after


def release(table, first, end, pool, page, capacity):
    """Pushes onto `pool` in place, up to `capacity`; an entry below 0 is no page."""
    for row, lo, hi in zip(table, first, end):
        for i, entry in enumerate(row):
            if lo <= i * page + page - 1 < hi and entry >= 0 and len(pool) < capacity:
                pool.append(entry)
