"""The paged cache's operators in numpy: 64-bit arithmetic, request by request."""
import numpy as np

from smith_amd.tensor import Tensor


def to_bf16(x):
    """f32 -> bf16 bits, nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def stored(x, dtype):
    """f32 values as a pool of dtype holds them (the host array of a Tensor)."""
    if dtype == "bf16":
        return to_bf16(x)
    return np.asarray(x, np.float32).astype(np.float16 if dtype == "f16" else np.float32)


def value(bits, dtype):
    """What a pool's host array stands for, in f64."""
    if dtype == "bf16":
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return bits.astype(np.float64)


def upload(a, dtype=None):
    a = np.ascontiguousarray(a)
    t = Tensor(list(a.shape), dtype or {"float32": "f32", "int32": "i32", "float16": "f16", "uint16": "bf16"}[a.dtype.name])
    return t.set_data(a)


def plan(cached, added, free, free_count, tables, P, max_rows):
    """(tables, rowStart, lens, slots, positions, freeLeft) one row at a time."""
    tables = tables.copy()
    row_start, slots, positions = [0], np.full(max_rows, -1, np.int32), np.full(max_rows, -1, np.int32)
    left = free_count
    for b in range(len(cached)):
        for i in range(added[b]):
            p = cached[b] + i
            if p % P == 0:
                left -= 1
                tables[b, p // P] = free[left]
            r = row_start[-1] + i
            positions[r] = p
            slots[r] = tables[b, p // P] * P + p % P
        row_start.append(row_start[-1] + added[b])
    return tables, np.array(row_start, np.int32), (cached + added).astype(np.int32), slots, positions, left


def rotate(x, pos, cos, sin, half):
    """Pairs (i, i + half) of the last axis, in f64."""
    at = pos[:, None] * half + np.arange(half)
    c, s = cos.astype(np.float64)[at], sin.astype(np.float64)[at]
    if x.ndim == 3:
        c, s = c[:, None], s[:, None]
    x = x.astype(np.float64)
    return np.concatenate([x[..., :half] * c - x[..., half:] * s, x[..., :half] * s + x[..., half:] * c], -1)


def gathered(pool, table, n):
    """Keys 0 .. n-1 of one request: [kv heads, n, head dim]."""
    P = pool.shape[2]
    pages = pool[table[:-(-n // P)]]
    return pages.transpose(1, 0, 2, 3).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def attention(q, row_start, lens, tables, k, v, scale=None):
    """(out, magnitude, largest score sum): rows of q [rows, heads, dim] f64 over
    pools of f64 values; magnitude = sum p |v| / sum p bounds the terms of an
    output, and the last [rows, heads] is max_t scale sum |q_e k_te|."""
    H, D = q.shape[1:]
    nKV = k.shape[1]
    G = H // nKV
    scale = D ** -0.5 if not scale else scale
    out, mag, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for b, n in enumerate(lens):
        r0, r1 = row_start[b], row_start[b + 1]
        if r0 == r1 or n == 0:
            continue
        kk, vv = gathered(k, tables[b], n), gathered(v, tables[b], n)
        for r in range(r0, r1):
            t = n - (r1 - r0) + (r - r0) + 1
            for h in range(H):
                kt, vt = kk[h // G, :t], vv[h // G, :t]
                s = scale * (kt @ q[r, h])
                p = np.exp(s - s.max())
                out[r, h] = p @ vt / p.sum()
                mag[r, h] = p @ np.abs(vt) / p.sum()
                big[r, h] = abs(scale) * (np.abs(kt) @ np.abs(q[r, h])).max()
    return out, mag, big
