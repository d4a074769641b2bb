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


def attention(q, row_start, lens, tables, k, v, seen, scale=None):
    """(out, magnitude, largest score sum, keys), as paged_reference.attention, of rows that
    see the keys for which seen(b, position, key numbers) holds: pools k, v of f64 values."""
    H, D = q.shape[1:]
    G, P = H // k.shape[1], k.shape[2]
    scale = D ** -0.5 if not scale else scale
    out, mag, big, keys = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(len(q))
    for b, n in enumerate(lens):
        r0, r1 = row_start[b], row_start[b + 1]
        for r in range(r0, r1):
            at = n - (r1 - r0) + (r - r0)
            t = np.arange(at + 1)
            t = t[seen(b, at, t)]
            keys[r] = len(t)
            if not len(t):
                continue
            page = tables[b][t // P]
            kk, vv = k[page, :, t % P], v[page, :, t % P]  # [keys, kv heads, dim]
            for h in range(H):
                kt, vt = kk[:, h // G], vv[:, h // G]
                s = scale * (kt @ q[r, h])
                p = np.exp(s - s.max())
                out[r, h] = p @ vt / p.sum()
                mag[r, h] = p @ np.abs(vt) / p.sum()
                big[r, h] = abs(scale) * (np.abs(kt) @ np.abs(q[r, h])).max()
    return out, mag, big, keys


def check_attention(got, want, D):
    """The bound of an output (one of f32, f16 or bf16 pages): a score is a sum of D
    products of q (kept to 2^-22 of its row's largest element) and k in f32: off by at
    most (D + 8) 2^-24 + 2^-21 of B = scale sum |q k|; its weight by twice that, and by
    2^-21 for the exponential and the weight's own split; the sums over n keys by n half
    steps, each relative to sum p |v| / sum p; a join of two such sums by 2^-21."""
    out, mag, big, keys = want
    rel = 2 * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) * big + 2.0 ** -20 + keys[:, None] * 2.0 ** -23 + 2.0 ** -21
    off = np.abs(got.astype(np.float64).reshape(out.shape) - out)
    assert np.all(off <= mag * rel[..., None]), (off / (mag * rel[..., None] + 1e-300)).max()
    norm = np.linalg.norm(out)
    if norm:
        assert np.linalg.norm(off) <= 1e-5 * norm, np.linalg.norm(off) / norm
