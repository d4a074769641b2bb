"""Fork and compact of a paged cache's pages in plain Python, entry by entry."""
import numpy as np


def kept(j, P, n, window, sinks):
    """Whether page j of a request of n keys has one that is a sink or that the row at position n sees."""
    keys = range(j * P, (j + 1) * P)
    return not window or any(k < sinks or k > n - window for k in keys)


def fork(lens, tables, parents, n_pages, P, new_tables, free, window=0, sinks=0):
    """(new lens, new tables, free list, its count, copies as (from, to, keys))."""
    new_lens, new_tables, free = np.zeros_like(lens), new_tables.copy(), free.copy()
    live, seen, waiting = set(), set(), []
    for b, p in enumerate(parents):
        if p < 0:
            continue
        n = int(lens[p])
        new_lens[b] = n
        for j in range(-(-n // P)):
            new_tables[b, j] = tables[p, j] if kept(j, P, n, window, sinks) else -1
            if new_tables[b, j] >= 0:
                live.add(int(new_tables[b, j]))
        if p in seen and n % P:
            waiting.append(b)
        seen.add(p)
    unused = [q for q in range(n_pages) if q not in live]
    copies = []
    for b in waiting:
        q, p = unused.pop(0), parents[b]
        copies.append((int(tables[p, lens[p] // P]), q, int(lens[p] % P)))
        new_tables[b, lens[p] // P] = q
    free[:len(unused)] = unused[::-1]
    return new_lens, new_tables, free, len(unused), copies


def compact(lens, tables, n_pages, P, free, window=0, sinks=0):
    """(new tables, free list, its count, moves as (from, to))."""
    tables, free = tables.copy(), free.copy()
    named = [(b, j) for b, n in enumerate(lens) for j in range(-(-int(n) // P))]
    live = sorted({int(tables[b, j]) for b, j in named if kept(j, P, int(lens[b]), window, sinks)})
    n = len(live)
    holes = [q for q in range(n) if q not in live]
    moves = list(zip([q for q in live if q >= n], holes))
    to = dict(moves)
    for b, j in named:
        q = int(tables[b, j])
        tables[b, j] = to.get(q, q) if kept(j, P, int(lens[b]), window, sinks) else -1
    free[:n_pages - n] = np.arange(n_pages - 1, n - 1, -1)
    return tables, free, n_pages - n, moves
