"""Workloads of several continuations of one prompt, bounded caches and scores.

  fork      smith_paged_fork: requests become continuations of others (or of
            none), share the full pages, get a copy of the partly filled one,
            and leave the free list of the pages that nobody names any more
  compact   smith_paged_compact: the live pages move to the pool's low end
  window    smith_paged_attention_window: a row sees the first `sinks` keys and
            the `window` keys up to its own
  shared    smith_paged_attention_shared: groups of requests have their first
            keys in common, whose attention is computed once a group
  logprobs  smith_logprobs: of rows of logits the log probabilities of given
            tokens, the entropy and the top alternatives

The pools are [pages][kv heads][page size][head dim] of f32, f16 or bf16; q and
the attention's outputs are f32.  Inputs come from the seed alone: pages in random
order, values N(0, 1) (queries N(0, 2): attention that has preferences).
"""
import ctypes
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2), "bf16": (2, torch.bfloat16, 2)}


def listed():
    return [
        # one prompt goes on in six ways: the smallest call, its latency
        {"name": "fork_1_to_6_f16", "op": "fork", "type": "f16", "layers": 4, "kv": 4, "dim": 64, "page": 16, "groups": 1,
         "width": 8, "shared": 700, "own": 0, "how": "fan", "window": 0, "sinks": 0},
        # a step of beam search: each group's beams go on from some of them
        {"name": "fork_beams_40x4_f16", "op": "fork", "type": "f16", "layers": 16, "kv": 4, "dim": 64, "page": 16,
         "groups": 40, "width": 4, "shared": 1500, "own": 90, "how": "beams", "window": 0, "sinks": 0},
        # half of a server's requests have ended: the pool before it is made smaller
        {"name": "compact_300_f32", "op": "compact", "type": "f32", "layers": 16, "kv": 4, "dim": 64, "page": 16,
         "groups": 100, "width": 3, "shared": 300, "own": 200, "how": "ended", "window": 0, "sinks": 0},
        # a few chats on a small model: latency
        {"name": "window_3x1200_f32", "op": "window", "type": "f32", "heads": 16, "kv": 4, "dim": 64, "page": 16,
         "reqs": 3, "longest": 1200, "spread": "near", "rows": 1, "window": 512, "sinks": 4},
        # a full server of long chats, the pages behind the window given back
        {"name": "window_64x30000_bf16", "op": "window", "type": "bf16", "heads": 32, "kv": 8, "dim": 128, "page": 32,
         "reqs": 64, "longest": 30000, "spread": "log", "rows": 1, "window": 4096, "sinks": 4},
        # a chunk of a long prompt
        {"name": "window_chunk_1500_f16", "op": "window", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "reqs": 1, "longest": 9000, "spread": "near", "rows": 1500, "window": 2048, "sinks": 64},
        # four answers to one question
        {"name": "shared_4x700_f32", "op": "shared", "type": "f32", "heads": 16, "kv": 4, "dim": 64, "page": 16,
         "groups": 1, "width": 4, "shared": 700, "own": 40, "rows": 1},
        # many requests behind one long instruction
        {"name": "shared_64x6001_f16", "op": "shared", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "groups": 1, "width": 64, "shared": 6001, "own": 300, "rows": 1},
        # groups of continuations of different prompts, a few drafted tokens each: the most arithmetic
        {"name": "shared_12x16_bf16", "op": "shared", "type": "bf16", "heads": 32, "kv": 8, "dim": 128, "page": 32,
         "groups": 12, "width": 16, "shared": 9000, "own": 500, "rows": 4},
        # the next token's alternatives
        {"name": "logprobs_1x32000_f32", "op": "logprobs", "type": "f32", "rows": 1, "vocab": 32000, "given": 1,
         "top": 5, "banned": 0.0},
        # a batch's, an odd vocabulary, some of it banned
        {"name": "logprobs_57x50003_bf16", "op": "logprobs", "type": "bf16", "rows": 57, "vocab": 50003, "given": 3,
         "top": 20, "banned": 0.01},
        # the scores of a text: the most bytes
        {"name": "logprobs_900x131072_f32", "op": "logprobs", "type": "f32", "rows": 900, "vocab": 131072, "given": 1,
         "top": 8, "banned": 0.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    r = rng.random()
    page = rng.choice([8, 16, 16, 32, 64, 128])
    kind = rng.choice(["f32", "f16", "bf16"])
    if r < 0.3:
        groups = _log_int(rng, 1, 120)
        case = {"op": rng.choice(["fork", "fork", "compact"]), "type": kind, "layers": _log_int(rng, 1, 24),
                "kv": rng.choice([1, 2, 4, 8]), "dim": rng.choice([40, 64, 80, 128]), "page": page, "groups": groups,
                "width": _log_int(rng, 1, max(1, 256 // groups)), "shared": _log_int(rng, 1, 2000),
                "own": rng.choice([0, _log_int(rng, 1, 250)]), "how": rng.choice(["fan", "beams", "ended"]),
                "window": 0, "sinks": 0}
        if case["op"] == "fork" and rng.random() < 0.3:
            case["window"], case["sinks"] = _log_int(rng, 1, 1000), rng.choice([0, rng.randint(1, 70)])
        room = 400e6 / (2 * case["kv"] * case["dim"] * (4 if kind == "f32" else 2))
        room /= groups * (case["shared"] + case["width"] * (case["own"] + page)) + page
        case["layers"] = max(1, min(case["layers"], int(room)))
        return case
    if r < 0.55:
        rows, vocab = _log_int(rng, 1, 2000), _log_int(rng, 1, 200000)
        return {"op": "logprobs", "type": kind, "rows": min(rows, max(1, 100000000 // vocab)), "vocab": vocab,
                "given": rng.choice([0, 1, 1, rng.randint(2, 9)]), "top": min(vocab, rng.choice([0, 1, rng.randint(2, 64)])),
                "banned": rng.choice([0.0, 0.0, rng.uniform(0.0, 0.5)])}
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 4, 64), (32, 4, 64), (16, 16, 128), (8, 1, 128), (9, 3, 64),
                                 (10, 2, 80), (12, 4, 96), (10, 10, 40)])
    case = {"type": kind, "heads": heads, "kv": kv, "dim": dim, "page": page}
    if r < 0.78:
        longest, window = _log_int(rng, 1, 40000), _log_int(rng, 1, 5000)
        rows = rng.choice([1, _log_int(rng, 1, min(longest, 1500))])
        seen = min(longest, window + rows)
        reqs = _log_int(rng, 1, max(1, min(128, 250000 // seen, 5000000 // (rows * seen))))
        return {"op": "window", **case, "reqs": reqs, "longest": longest, "spread": rng.choice(["near", "log"]),
                "rows": rows, "window": window, "sinks": rng.choice([0, 4, rng.randint(1, 200)])}
    shared, rows = _log_int(rng, 1, 12000), rng.choice([1, 1, rng.randint(2, 6)])
    width = _log_int(rng, 1, max(1, min(128, 1500000 // (shared * rows))))
    groups = _log_int(rng, 1, max(1, min(192 // width, 100000 // shared)))
    return {"op": "shared", **case, "groups": groups, "width": width, "shared": shared,
            "own": _log_int(rng, rows, 500), "rows": rows}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 7919 + salt) % (1 << 62))
    return g


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _full(shape, value, dtype=torch.int32):
    return torch.full(shape, value, device=DEV, dtype=dtype)


def _pool(case, shape, seed, salt):
    return torch.randn(*shape, case["kv"], case["page"], case["dim"], generator=_gen(seed, salt), device=DEV,
                       dtype=TYPES[case["type"]][1])


def _shared_lengths(case):
    """(shared [groups], lens [requests]): the same for every seed.  A prompt's
    length is `shared` or, of the later groups, less; a request adds up to `own`."""
    rs = np.random.RandomState(case["groups"] * 1000 + case["width"])
    n, least = case["groups"] * case["width"], case.get("rows", 0)
    shared = np.exp(rs.uniform(math.log(max(1, case["shared"] // 4)), math.log(case["shared"] + 1), case["groups"]))
    shared = shared.astype(np.int64).clip(1, case["shared"])
    shared[0] = case["shared"]
    more = rs.randint(least, max(least, case["own"]) + 1, n)
    more[0] = max(least, case["own"])
    return shared, shared.repeat(case["width"]) + more


def _shared_tables(rs, P, width, shared, lens, spare):
    """Block tables in which the requests of a group name the same pages for the
    full pages of their shared keys, and pages of their own behind them; the
    number of pages, `spare` of them in nobody's table."""
    full, pages = (shared // P).repeat(width), -(-lens // P)
    mine = pages - full
    n_pages = int((shared // P).sum() + mine.sum()) + spare
    order = rs.permutation(n_pages)
    of_group = np.concatenate([[0], np.cumsum(shared // P)])
    first = of_group[-1] + np.concatenate([[0], np.cumsum(mine)])
    j = np.arange(int(pages.max()) + 2)[None, :]
    at = np.where(j < full[:, None], of_group[:-1].repeat(width)[:, None] + j, first[:-1, None] + j - full[:, None])
    return np.where(j < pages[:, None], order[at.clip(0, n_pages - 1)], -1), n_pages


def _prepare_fork(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    P, width, n = case["page"], case["width"], case["groups"] * case["width"]
    shared, lens = _shared_lengths(case)
    if case["how"] == "fan":  # the groups' other places are empty as yet
        lens = np.where(np.arange(n) % width == 0, lens, 0)
        tables, n_pages = _shared_tables(rs, P, width, shared * 0, lens, n + 3)
    else:
        tables, n_pages = _shared_tables(rs, P, width, shared, lens, n + 3)
    first = np.arange(n) // width * width
    if case["how"] == "fan":
        parents = np.where(np.arange(n) % width < max(1, width * 3 // 4), first, -1)
    elif case["how"] == "beams":
        parents = first + rs.randint(0, width, n)
    else:  # half of the groups have ended
        parents = np.where((rs.permutation(case["groups"]) % 2).astype(bool)[np.arange(n) // width], np.arange(n), -1)
    if case["op"] == "compact":
        lens = np.where(parents >= 0, lens, 0)
    st = {"lens": _i32(lens), "tables": _i32(tables), "parents": _i32(parents), "n_pages": n_pages,
          "pools": _pool(case, (2 * case["layers"], n_pages), seed, 2), "new_lens": _full((n,), 0),
          "new_tables": _full(tables.shape, -2), "free": _full((n_pages,), -2), "free_count": _full((1,), 0)}
    st["pointers"] = (ctypes.c_void_p * len(st["pools"]))(*[p.data_ptr() for p in st["pools"]])
    return st


def _window_lengths(case):
    """(lens, rows that each request brings): the same for every seed."""
    rs = np.random.RandomState(case["reqs"])
    n, longest = case["reqs"], case["longest"]
    if case["spread"] == "near":
        lens = rs.randint(max(1, longest * 7 // 10), longest + 1, n)
    else:
        lens = np.exp(rs.uniform(0, math.log(longest + 1), n)).astype(np.int64).clip(1, longest)
    lens[0] = longest
    added = np.where(rs.rand(n) < 0.5, 1, rs.randint(1, case["rows"] + 1, n))
    added[0] = case["rows"]
    return lens, np.minimum(added, lens)


def _prepare_window(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    P, W, S = case["page"], case["window"], case["sinks"]
    lens, added = _window_lengths(case)
    order = rs.permutation(case["reqs"])
    lens, added = lens[order], added[order]
    # pages with a key that some row sees; the others were given back
    j = np.arange(-(-int(lens.max()) // P) + 1)[None, :]
    kept = (j * P < lens[:, None]) & ((j * P < S) | ((j + 1) * P > (lens - added + 1 - W)[:, None]))
    n_pages = int(kept.sum()) + 2
    tables = np.full(kept.shape, -1)
    tables[kept] = rs.permutation(n_pages)[:int(kept.sum())]
    rows, width = int(added.sum()), case["heads"] * case["dim"]
    return {"q": torch.randn(rows, width, generator=_gen(seed, 1), device=DEV) * 2.0, "tables": _i32(tables),
            "lens": _i32(lens), "row_start": None if case["rows"] == 1 else _i32(np.concatenate([[0], np.cumsum(added)])),
            "k": _pool(case, (n_pages,), seed, 2), "v": _pool(case, (n_pages,), seed, 3), "rows": rows,
            "most_added": int(added.max()), "out": _full((rows, width), 3.0, torch.float32)}


def _prepare_shared(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    P, width, n = case["page"], case["width"], case["groups"] * case["width"]
    shared, lens = _shared_lengths(case)
    tables, n_pages = _shared_tables(rs, P, width, shared, lens, 2)
    added = np.random.RandomState(n).randint(1, case["rows"] + 1, n)
    added[0] = case["rows"]
    rows, cols = int(added.sum()), case["heads"] * case["dim"]
    st = {"q": torch.randn(rows, cols, generator=_gen(seed, 1), device=DEV) * 2.0, "tables": _i32(tables),
          "lens": _i32(lens), "row_start": None if case["rows"] == 1 else _i32(np.concatenate([[0], np.cumsum(added)])),
          "group_start": _i32(np.arange(case["groups"] + 1) * width), "shared": _i32(shared),
          "longest_shared": int(shared.max()), "longest_own": int((lens - shared.repeat(width)).max()),
          "k": _pool(case, (n_pages,), seed, 2), "v": _pool(case, (n_pages,), seed, 3), "rows": rows,
          "most_added": int(added.max()), "out": _full((rows, cols), 3.0, torch.float32)}
    # the shared keys of a partly filled page are in each request's own page
    for g in np.nonzero(shared % P)[0]:
        at, part = shared[g] // P, shared[g] % P
        to = st["tables"][g * width + 1:(g + 1) * width, at].long()
        for pool in (st["k"], st["v"]):
            pool[to, :, :part] = pool[int(tables[g * width, at]), :, :part].clone()
    return st


def _prepare_logprobs(case, seed):
    rows, vocab, given, top = case["rows"], case["vocab"], case["given"], case["top"]
    g = _gen(seed, 1)
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.5
    if case["banned"]:
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device=DEV) < case["banned"], -math.inf)
    return {"logits": x.to(TYPES[case["type"]][1]),
            "tokens": torch.randint(0, vocab, (rows, given), generator=g, device=DEV, dtype=torch.int32) if given else None,
            "logprobs": _full((rows, given), 3.0, torch.float32), "entropy": _full((rows,), 3.0, torch.float32),
            "top_ids": _full((rows, top), -2), "top_logprobs": _full((rows, top), 3.0, torch.float32)}


def prepare(case, seed):
    st = {"fork": _prepare_fork, "compact": _prepare_fork, "window": _prepare_window, "shared": _prepare_shared,
          "logprobs": _prepare_logprobs}[case["op"]](case, seed)
    st["case"] = case
    return st


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _kept(st, lens):
    """[requests][pages of a table]: there, and with a key that a later row sees."""
    c = st["case"]
    P, j = c["page"], torch.arange(st["tables"].shape[1], device=DEV)[None, :]
    there = j * P < lens[:, None]
    if not c["window"]:
        return there, there
    return there, there & ((j * P < c["sinks"]) | ((j + 1) * P > lens[:, None] + 1 - c["window"]))


def _plain_fork(st):
    P, n = st["case"]["page"], len(st["lens"])
    parents, b = st["parents"].long(), torch.arange(n, device=DEV)
    p = parents.clamp(min=0)
    lens = torch.where(parents >= 0, st["lens"].long()[p], 0)
    there, kept = _kept(st, lens)
    tables = torch.where(kept, st["tables"][p], -1)
    first = torch.full((n + 1,), n, device=DEV).scatter_reduce(0, torch.where(parents >= 0, p, n), b, "amin")[p]
    copies = torch.nonzero((lens % P > 0) & (first != b))[:, 0]
    last = lens[copies] // P
    live = torch.zeros(st["n_pages"], dtype=torch.bool, device=DEV)
    live[tables[kept].long()] = True
    free = torch.nonzero(~live)[:, 0].int()
    src, dst = tables[copies, last].long(), free[:len(copies)].long()
    tables[copies, last] = dst.int()
    used = (torch.arange(P, device=DEV)[None, :] < (lens[copies] % P)[:, None])[None, :, None, :, None]
    st["pools"][:, dst] = torch.where(used, st["pools"][:, src], st["pools"][:, dst])
    rest = free[len(copies):].flip(0)
    st["free"][:len(rest)] = rest
    return {"lens": lens.int(), "tables": torch.where(there, tables, st["new_tables"]), "free": st["free"],
            "free_count": _full((1,), len(rest)), "pools": st["pools"]}


def _plain_compact(st):
    there, _ = _kept(st, st["lens"].long())
    live = torch.zeros(st["n_pages"], dtype=torch.bool, device=DEV)
    live[st["tables"][there].long()] = True
    n = int(live.sum())
    src, dst = torch.nonzero(live[n:])[:, 0] + n, torch.nonzero(~live[:n])[:, 0]
    now = torch.arange(st["n_pages"], device=DEV, dtype=torch.int32)
    now[src] = dst.int()
    st["pools"][:, dst] = st["pools"][:, src]
    left = st["n_pages"] - n
    st["free"][:left] = torch.arange(st["n_pages"] - 1, n - 1, -1, device=DEV, dtype=torch.int32)
    return {"tables": torch.where(there, now[st["tables"].clamp(min=0).long()], st["new_tables"]), "free": st["free"],
            "free_count": _full((1,), left), "pools": st["pools"]}


def _keys(pool, tables, at):
    """Keys at positions at [requests, n] of the requests in f32: [requests, kv heads, n, dim]."""
    P = pool.shape[2]
    page = tables.long().gather(1, (at // P).clamp(max=tables.shape[1] - 1)).clamp(min=0)
    return pool[page, :, at % P].transpose(1, 2).float()


def _padded(st, n):
    """q as [requests, most rows, kv heads, heads of each, dim] and the rows' positions [requests, most rows]."""
    c = st["case"]
    G = c["heads"] // c["kv"]
    lens = st["lens"].long()
    start = torch.arange(n + 1, device=DEV) if st["row_start"] is None else st["row_start"].long()
    i = torch.arange(st["most_added"], device=DEV)
    q = st["q"][(start[:-1, None] + i).clamp(max=st["rows"] - 1)].view(n, st["most_added"], c["kv"], G, c["dim"])
    return q, (lens - start[1:] + start[:-1])[:, None] + i, start


def _rows(st, o, start, n):
    """Rows of o [requests, most rows, width] side by side."""
    r = torch.arange(st["rows"], device=DEV)
    b = torch.searchsorted(start[1:], r, right=True)
    st["out"].copy_(o.reshape(n * st["most_added"], -1)[b * st["most_added"] + r - start[b]])
    return st["out"]


def _plain_window(st):
    c = st["case"]
    H, Hk, D, W, S, n, most = c["heads"], c["kv"], c["dim"], c["window"], c["sinks"], c["reqs"], st["most_added"]
    G, lens = H // Hk, st["lens"].long()
    q, at, start = _padded(st, n)
    # the sinks, and as many keys behind them as some row may see, up to the end
    wide = min(c["longest"], W + most - 1)
    t = torch.cat([torch.arange(S, device=DEV).expand(n, S), lens[:, None] - wide + torch.arange(wide, device=DEV)], 1)
    first = torch.arange(t.shape[1], device=DEV) < S
    k, v = _keys(st["k"], st["tables"], t.clamp(min=0)), _keys(st["v"], st["tables"], t.clamp(min=0))
    seen = (t[:, None] <= at[:, :, None]) & torch.where(first, t[:, None] < S, (t[:, None] >= S) & (t[:, None] > at[:, :, None] - W))
    q = q.permute(0, 2, 1, 3, 4).reshape(n, Hk, most * G, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    s = s.masked_fill(~seen.repeat_interleave(G, 1)[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return _rows(st, o.view(n, Hk, most, G, D).permute(0, 2, 1, 3, 4).reshape(n, most, H * D), start, n)


def _plain_shared(st):
    c = st["case"]
    H, Hk, D, groups, width, most = c["heads"], c["kv"], c["dim"], c["groups"], c["width"], st["most_added"]
    G, n, shared = H // Hk, groups * width, st["shared"].long()
    q, at, start = _padded(st, n)
    # a group's columns against its shared keys, its first request's
    t = torch.arange(st["longest_shared"], device=DEV).expand(groups, -1)
    firsts = st["tables"][::width]
    k, v = _keys(st["k"], firsts, t), _keys(st["v"], firsts, t)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, Hk, most * G, D)
    qg = q.view(groups, width, Hk, most * G, D).transpose(1, 2).reshape(groups, Hk, width * most * G, D)
    s = torch.matmul(qg, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    s = s.masked_fill((t >= shared[:, None])[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    l, o = p.sum(-1, keepdim=True), torch.matmul(p, v)
    del s, p

    def by_request(x):
        return x.view(groups, Hk, width, most * G, -1).transpose(1, 2).reshape(n, Hk, most * G, -1)

    m, l, o = by_request(m), by_request(l), by_request(o)
    # each request's against its own
    t = shared.repeat_interleave(width)[:, None] + torch.arange(st["longest_own"], device=DEV)
    k, v = _keys(st["k"], st["tables"], t), _keys(st["v"], st["tables"], t)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    s = s.masked_fill((t[:, None] > at[:, :, None]).repeat_interleave(G, 1)[:, None], -math.inf)
    both = torch.maximum(m, s.amax(-1, keepdim=True))
    p, f = torch.exp(s - both), torch.exp(m - both)
    o = (o * f + torch.matmul(p, v)) / (l * f + p.sum(-1, keepdim=True))
    return _rows(st, o.view(n, Hk, most, G, D).permute(0, 2, 1, 3, 4).reshape(n, most, H * D), start, n)


def _plain_logprobs(st):
    c = st["case"]
    x = st["logits"].float()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    l = e.sum(1, keepdim=True)
    log_l = torch.log(l)
    entropy = (log_l - (e * torch.where(e > 0, d, 0.0)).sum(1, keepdim=True) / l)[:, 0]
    out = {"entropy": entropy, "logprobs": d.gather(1, st["tokens"].long()) - log_l if c["given"] else st["logprobs"]}
    # equal values in the order of their places: value and place as one whole number
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
    order = (bits << 32) + (c["vocab"] - torch.arange(c["vocab"], device=DEV))
    ids = order.topk(c["top"], 1).indices
    return {**out, "top_ids": ids.int(), "top_logprobs": d.gather(1, ids) - log_l}


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------
def _own_fork(st):
    from smith_amd import device
    c = st["case"]
    n, max_pages = st["tables"].shape
    device.check(device.lib.smith_paged_fork(
        device.ops_ctx(), TYPES[c["type"]][0], st["lens"].data_ptr(), st["tables"].data_ptr(), st["parents"].data_ptr(),
        n, max_pages, c["window"], c["sinks"], c["kv"], c["dim"], st["pointers"], len(st["pools"]), st["n_pages"],
        c["page"], st["new_lens"].data_ptr(), st["new_tables"].data_ptr(), st["free"].data_ptr(),
        st["free_count"].data_ptr()), "fork")
    return {"lens": st["new_lens"], "tables": st["new_tables"], "free": st["free"], "free_count": st["free_count"],
            "pools": st["pools"]}


def _own_compact(st):
    from smith_amd import device
    c = st["case"]
    n, max_pages = st["tables"].shape
    device.check(device.lib.smith_paged_compact(
        device.ops_ctx(), TYPES[c["type"]][0], st["lens"].data_ptr(), st["tables"].data_ptr(), n, max_pages, c["window"],
        c["sinks"], c["kv"], c["dim"], st["pointers"], len(st["pools"]), st["n_pages"], c["page"],
        st["new_tables"].data_ptr(), st["free"].data_ptr(), st["free_count"].data_ptr()), "compact")
    return {"tables": st["new_tables"], "free": st["free"], "free_count": st["free_count"], "pools": st["pools"]}


def _own_window(st):
    from smith_amd import device
    c = st["case"]
    width, start = st["q"].shape[1], st["row_start"]
    device.check(device.lib.smith_paged_attention_window(
        device.ops_ctx(), TYPES[c["type"]][0], st["q"].data_ptr(), width, st["rows"],
        start.data_ptr() if start is not None else None, st["lens"].data_ptr(), st["tables"].data_ptr(), c["reqs"],
        st["tables"].shape[1], c["window"], c["sinks"], c["heads"], c["kv"], c["dim"], 0.0, st["k"].data_ptr(),
        st["v"].data_ptr(), st["k"].shape[0], c["page"], st["out"].data_ptr(), width), "attention")
    return st["out"]


def _own_shared(st):
    from smith_amd import device
    c = st["case"]
    width, start = st["q"].shape[1], st["row_start"]
    device.check(device.lib.smith_paged_attention_shared(
        device.ops_ctx(), TYPES[c["type"]][0], st["q"].data_ptr(), width, st["rows"],
        start.data_ptr() if start is not None else None, st["lens"].data_ptr(), st["tables"].data_ptr(),
        len(st["lens"]), st["tables"].shape[1], st["group_start"].data_ptr(), st["shared"].data_ptr(), c["groups"],
        c["heads"], c["kv"], c["dim"], 0.0, st["k"].data_ptr(), st["v"].data_ptr(), st["k"].shape[0], c["page"],
        st["out"].data_ptr(), width), "attention")
    return st["out"]


def _own_logprobs(st):
    from smith_amd import device
    c = st["case"]
    device.check(device.lib.smith_logprobs(
        device.ops_ctx(), TYPES[c["type"]][0], st["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"],
        st["tokens"].data_ptr() if c["given"] else None, c["given"], c["top"], st["logprobs"].data_ptr() if c["given"] else None,
        st["entropy"].data_ptr(), st["top_ids"].data_ptr() if c["top"] else None,
        st["top_logprobs"].data_ptr() if c["top"] else None), "logprobs")
    return {name: st[name] for name in ("entropy", "logprobs", "top_ids", "top_logprobs")}


def run(st):
    op = st["case"]["op"]
    if own:
        return {"fork": _own_fork, "compact": _own_compact, "window": _own_window, "shared": _own_shared,
                "logprobs": _own_logprobs}[op](st)
    return {"fork": _plain_fork, "compact": _plain_compact, "window": _plain_window, "shared": _plain_shared,
            "logprobs": _plain_logprobs}[op](st)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _work_fork(case):
    P, width, n = case["page"], case["width"], case["groups"] * case["width"]
    shared, lens = _shared_lengths(case)
    if case["how"] == "fan":
        lens = np.where(np.arange(n) % width == 0, lens, 0)
    key = 2 * case["layers"] * case["kv"] * case["dim"] * TYPES[case["type"]][2]
    pages = -(-lens // P)
    mine = int((pages - (shared // P).repeat(width)).sum())
    total = int((shared // P).sum()) + mine if case["how"] != "fan" else int(pages.sum())
    if case["op"] == "compact":  # the live pages of about half of the groups, half of those above the line
        left = total // 2
        return {"bytes": 8 * int(pages.sum()) // 2 + 4 * (total - left) + left // 2 * P * key * 2, "flops": 0}
    if case["how"] == "fan":
        children = max(1, width * 3 // 4)
        copied = int((lens % P).sum()) * (children - 1)
        entries = int(pages.sum()) * (1 + children)
    elif case["how"] == "beams":  # a beam goes on in one way on average, in none with probability (1 - 1/w)^w
        copied = int((lens % P).mean() * n * (1 - 1 / width) ** width)
        entries = 2 * int(pages.sum())
    else:
        copied, entries = 0, int(pages.sum())
    return {"bytes": 4 * entries + 12 * n + 4 * (n + 3) + 2 * copied * key, "flops": 0}


def work(case):
    if case["op"] in ("fork", "compact"):
        return _work_fork(case)
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * TYPES[case["type"]][2] + case["rows"] * (8 * case["given"] + 8 * case["top"] + 4), "flops": 6.0 * n}
    H, Hk, D, P, e = case["heads"], case["kv"], case["dim"], case["page"], TYPES[case["type"]][2]
    if case["op"] == "window":
        lens, added = _window_lengths(case)
        W, S = case["window"], case["sinks"]
        union = np.minimum(lens, W + added - 1)  # keys that some row sees behind the sinks, or with them
        union += np.minimum(S, lens - union)
        keys = sum(int(np.minimum(np.arange(n - a + 1, n + 1), W + S).sum()) for n, a in zip(lens, added))
        return {"bytes": int(union.sum()) * 2 * Hk * D * e + int(added.sum()) * 8 * H * D + 4 * int((-(-union // P)).sum()),
                "flops": 4.0 * H * D * keys}
    shared, lens = _shared_lengths(case)
    n = len(lens)
    added = np.random.RandomState(n).randint(1, case["rows"] + 1, n)
    added[0] = case["rows"]
    alone = int(shared.sum()) + int((lens - shared.repeat(case["width"])).sum())
    keys = (lens * added - added * (added - 1) // 2).sum()
    return {"bytes": alone * 2 * Hk * D * e + int(added.sum()) * 8 * H * D + 4 * (alone // P + n), "flops": 4.0 * H * D * float(keys)}


# --------------------------------------------------------------------------
# from the definitions in 64 bits, request by request
# --------------------------------------------------------------------------
def _exact_attention(case, seed):
    st = prepare(case, seed)
    H, Hk, D, P = case["heads"], case["kv"], case["dim"], case["page"]
    G, lens = H // Hk, st["lens"].tolist()
    W, S = case.get("window", 0), case.get("sinks", 0)
    start = st["row_start"].tolist() if st["row_start"] is not None else list(range(len(lens) + 1))
    out = torch.empty(st["rows"], H, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        r0, r1 = start[b], start[b + 1]
        at = torch.arange(n - (r1 - r0), n, device=DEV)[:, None]
        t = torch.arange(n, device=DEV)
        if W:
            t = t[(t < S) | (t > int(at[0, 0]) - W)]
        seen = t[None] <= at
        if W:
            seen &= (t[None] > at - W) | (t[None] < S)
        page = st["tables"][b].long()[t // P]
        q = st["q"][r0:r1].double().view(r1 - r0, H, D)
        for h in range(Hk):
            k, v = st["k"][page, h, t % P].double(), st["v"][page, h, t % P].double()
            x = q[:, h * G:(h + 1) * G].reshape(-1, D) @ k.T.contiguous() / D ** 0.5
            w = torch.where(seen.repeat_interleave(G, 0), x, -math.inf).softmax(1)
            out[r0:r1, h * G:(h + 1) * G] = (w @ v).view(r1 - r0, G, D)
    return out.view(st["rows"], H * D)


def _exact_logprobs(case, seed):
    st = _prepare_logprobs(case, seed)
    x = st["logits"].double().log_softmax(1)
    entropy = -torch.xlogy(x.exp(), x.exp()).sum(1)
    top = st["logits"].double().sort(1, descending=True).values[:, :case["top"]]
    shift = x.amax(1, keepdim=True) - st["logits"].double().amax(1, keepdim=True)
    return {"entropy": entropy, "logprobs": x.gather(1, st["tokens"].long()) if case["given"] else None, "top_ids": None,
            "top_logprobs": top + shift}


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers and copies: the plain form's have to be met
    return (_exact_logprobs if case["op"] == "logprobs" else _exact_attention)(case, seed)
