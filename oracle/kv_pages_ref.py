"""Pages of the block-scaled KV cache on the host, in numpy, one entry at a time: the oracle of scratch_llm_amd/quant/kv_pages.py.

A pool is [k_codes, v_codes, k_scale, v_scale] with the page as the second axis; tables, lengths and refs are int arrays,
changed in place."""

from __future__ import annotations

import numpy as np


def copy(pool, src, dst) -> None:
    pages = pool[0].shape[1]
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages:
            for x in pool:
                x[:, d] = x[:, s]


def _valid(page, pages) -> bool:
    return 0 <= page < pages


def _lowest(refs, n):
    free = np.flatnonzero(refs == 0)
    return None if len(free) < n else [int(p) for p in free[:n]]


def fork(parents, pool, table, lengths, refs, block) -> int:
    rows, width = table.shape
    pages = len(refs)
    new_table, new_lengths, new_refs = table.copy(), lengths.copy(), refs.copy()
    waiting = []
    for b, p in enumerate(parents):
        if p == b:
            continue
        entries, n = [-1] * width, 0
        if 0 <= p < rows:
            n = min(max(int(lengths[p]), 0), width * block)
            for j in range((n + block - 1) // block):
                entries[j] = int(table[p, j]) if _valid(table[p, j], pages) else -1
            if n % block and (parents[p] == p or p in list(parents[:b])):
                j = n // block
                if entries[j] >= 0:
                    waiting.append((b, j, entries[j]))
                entries[j] = -1
        for x in table[b]:
            if _valid(x, pages):
                new_refs[x] -= 1
        for x in entries:
            if x >= 0:
                new_refs[x] += 1
        new_table[b], new_lengths[b] = entries, n
    free = _lowest(new_refs, len(waiting))
    if free is None:
        return 0
    for (b, j, s), d in zip(waiting, free):
        new_table[b, j] = d
        new_refs[d] = 1
        copy(pool, [s], [d])
    table[...], lengths[...], refs[...] = new_table, new_lengths, new_refs
    return 1


def reserve(pool, table, starts, counts, refs, block) -> int:
    width, pages = table.shape[1], len(refs)
    wanted = []
    for b, (s, c) in enumerate(zip(starts, counts)):
        end = min(int(s) + max(int(c), 0), width * block)
        if s < 0 or end <= s:
            continue
        for j in range(s // block, (end + block - 1) // block):
            page = int(table[b, j])
            if not _valid(page, pages):
                wanted.append((b, j, -1))
            elif refs[page] > 1:
                wanted.append((b, j, page))
    free = _lowest(refs, len(wanted))
    if free is None:
        return 0
    for (b, j, s), d in zip(wanted, free):
        table[b, j] = d
        refs[d] = 1
        if s >= 0:
            refs[s] -= 1
            copy(pool, [s], [d])
    return 1


def free(keep, table, lengths, refs, block) -> None:
    for b, k in enumerate(keep):
        k = max(int(k), 0)
        lengths[b] = min(lengths[b], k)
        for j in range((k + block - 1) // block, table.shape[1]):
            if _valid(table[b, j], len(refs)):
                refs[table[b, j]] -= 1
            table[b, j] = -1


def compact(pool, table, refs):
    used = refs > 0
    live = int(used.sum())
    moved = np.where(used, np.arange(len(refs)), -1).astype(np.int32)
    src = [p for p in range(live, len(refs)) if used[p]]
    dst = [p for p in range(live) if not used[p]]
    copy(pool, src, dst)
    for s, d in zip(src, dst):
        moved[s], refs[d], refs[s] = d, refs[s], 0
    for b in range(table.shape[0]):
        for j in range(table.shape[1]):
            if _valid(table[b, j], len(refs)):
                table[b, j] = moved[table[b, j]]
    return live, moved
