"""Workloads of the paged key-value cache: several requests served at once.

  plan       smith_paged_plan: block tables, slots and positions of a step's
             rows from the requests' lengths
  append     smith_paged_append: rotary positions, then k and v of the rows
             into their slots of the page pools
  attention  smith_paged_attention: rows of ragged requests over the pages that
             their tables name; one new token a request, or the rows of prompts
             and of prompt chunks behind a cache

The pools are [pages][kv heads][page size][head dim] of f32, f16 or bf16; q, k,
v and the outputs are f32.  Inputs come from the seed alone: pages in random
order, values N(0, 1) (queries N(0, 2): attention that has preferences).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2), "bf16": (2, torch.bfloat16, 2)}
ROPES = {"none": 0, "row": 1, "head": 2}


def listed():
    return [
        # one decode step of a few chats: the smallest plan
        {"name": "plan_decode_24", "op": "plan", "reqs": 24, "page": 16, "longest": 2000, "most_added": 1, "spare_rows": 8},
        # prompts, chunks and decode rows of a full server in one step
        {"name": "plan_mixed_700", "op": "plan", "reqs": 700, "page": 32, "longest": 8000, "most_added": 129, "spare_rows": 77},
        # the rows of a decode step, some of the batch's places empty
        {"name": "append_decode_64", "op": "append", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "rows": 57,
         "spare_rows": 7, "page": 16, "rope": "head", "longest": 4000},
        # one prompt chunk as this framework's Llama files run it: f32 cache, whole-row rotary
        {"name": "append_chunk_256_f32", "op": "append", "type": "f32", "heads": 16, "kv": 4, "dim": 64, "rows": 256,
         "spare_rows": 0, "page": 32, "rope": "row", "longest": 700},
        # several prompts at once
        {"name": "append_prompts_6001", "op": "append", "type": "bf16", "heads": 32, "kv": 8, "dim": 128, "rows": 6001,
         "spare_rows": 0, "page": 64, "rope": "head", "longest": 8000},
        # one chat on a small model: latency
        {"name": "decode_1x517_f32", "op": "attention", "type": "f32", "heads": 16, "kv": 4, "dim": 64, "reqs": 1,
         "page": 16, "longest": 517, "spread": "near", "rows": 1},
        # a batch of chats of very different lengths
        {"name": "decode_32_ragged_f16", "op": "attention", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "reqs": 32,
         "page": 16, "longest": 6000, "spread": "log", "rows": 1},
        # one long document
        {"name": "decode_1x131071_f16", "op": "attention", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "reqs": 1,
         "page": 64, "longest": 131071, "spread": "near", "rows": 1},
        # a full server: the most bytes
        {"name": "decode_120x4000_bf16", "op": "attention", "type": "bf16", "heads": 32, "kv": 8, "dim": 128,
         "reqs": 120, "page": 32, "longest": 4000, "spread": "near", "rows": 1},
        # four prompts from empty caches
        {"name": "prompts_4x500_f16", "op": "attention", "type": "f16", "heads": 32, "kv": 8, "dim": 128, "reqs": 4,
         "page": 16, "longest": 611, "spread": "near", "rows": 611},
        # a chunk of a long prompt behind its cache: the most arithmetic
        {"name": "chunk_2000_of_8000_bf16", "op": "attention", "type": "bf16", "heads": 32, "kv": 8, "dim": 128,
         "reqs": 1, "page": 64, "longest": 8000, "spread": "near", "rows": 2000},
        # a mixed step: decode rows and short chunks, a head dim that is no power of two, no grouping of heads
        {"name": "mixed_20_f32", "op": "attention", "type": "f32", "heads": 10, "kv": 10, "dim": 80, "reqs": 20,
         "page": 8, "longest": 1500, "spread": "log", "rows": 77},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    page = rng.choice([8, 16, 16, 32, 64, 128])
    r = rng.random()
    if r < 0.2:
        reqs = _log_int(rng, 1, 1500)
        added = rng.choice([1, _log_int(rng, 1, max(2, 65536 // reqs))])
        return {"op": "plan", "reqs": reqs, "page": page, "longest": _log_int(rng, max(2, added), 16000),
                "most_added": added, "spare_rows": rng.choice([0, rng.randint(1, 100)])}
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 4, 64), (32, 4, 64), (16, 16, 128), (8, 1, 128), (9, 3, 64),
                                 (10, 2, 80), (12, 4, 96), (10, 10, 40)])
    case = {"type": rng.choice(["f32", "f16", "bf16"]), "heads": heads, "kv": kv, "dim": dim, "page": page}
    if r < 0.4:
        rope = rng.choice(["none", "row", "head", "head"])
        return {"op": "append", **case, "rows": _log_int(rng, 1, 6000), "spare_rows": rng.choice([0, rng.randint(1, 40)]),
                "rope": rope, "longest": _log_int(rng, 10, 1500 if rope == "row" else 16000)}
    if r < 0.75:
        longest = _log_int(rng, 1, 131071)
        reqs = _log_int(rng, 1, max(1, min(256, 400000 // longest)))
        return {"op": "attention", **case, "reqs": reqs, "longest": longest, "spread": rng.choice(["near", "log"]),
                "rows": 1}
    longest = _log_int(rng, 2, 8000)
    rows = _log_int(rng, 2, min(longest, 2000))
    reqs = _log_int(rng, 1, max(1, min(64, 6000000 // (rows * longest))))
    return {"op": "attention", **case, "reqs": reqs, "longest": longest, "spread": rng.choice(["near", "log"]),
            "rows": rows}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 7919 + salt) % (1 << 62))
    return g


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _spread(rs, n, longest, how):
    """n lengths up to `longest`, the first of them that long."""
    if how == "near":
        v = rs.randint(max(1, longest * 7 // 10), longest + 1, n)
    else:
        v = np.exp(rs.uniform(0, math.log(longest + 1), n)).astype(np.int64).clip(1, longest)
    v[0] = longest
    return v


def _tables(rs, pages, n_pages, spare):
    """Block tables [reqs][most pages + spare] of pages[b] pages each out of
    n_pages in random order, and the pages that are left."""
    order = rs.permutation(n_pages)
    first = np.concatenate([[0], np.cumsum(pages)])
    j = np.arange(int(pages.max()) + spare)[None, :]
    at = np.minimum(first[:-1, None] + j, n_pages - 1)
    return np.where(j < pages[:, None], order[at], 0), order[first[-1]:]


def _pool(case, n_pages, seed, salt):
    return torch.randn(n_pages, case["kv"], case["page"], case["dim"], generator=_gen(seed, salt), device=DEV,
                       dtype=TYPES[case["type"]][1])


def _plan_lengths(case, seed):
    """(random state, cached, added): the same lengths for every seed, in an order of the seed's."""
    rs = np.random.RandomState(case["reqs"])
    n, most = case["reqs"], case["most_added"]
    if most == 1:
        added = (rs.rand(n) < 0.9).astype(np.int64)
    else:
        added = np.where(rs.rand(n) < 0.5, 1, np.exp(rs.uniform(0, math.log(most + 1), n)).astype(np.int64).clip(0, most))
    cached = (_spread(rs, n, case["longest"], "log") - added).clip(0)
    rs = np.random.RandomState(seed % (1 << 32))
    order = rs.permutation(n)
    return rs, cached[order], added[order]


def _prepare_plan(case, seed):
    rs, cached, added = _plan_lengths(case, seed)
    P = case["page"]
    old, new = -(-cached // P), -(-(cached + added) // P)
    n_pages = int(new.sum()) + 5
    tables, free = _tables(rs, old, n_pages, int(new.max() - old.max()) + 3)
    rows = int(added.sum()) + case["spare_rows"] + 1
    n = case["reqs"]
    return {"cached": _i32(cached), "added": _i32(added), "free": _i32(free), "free_count": _i32([len(free)]),
            "tables": _i32(tables), "n_pages": n_pages, "rows": rows, "max_rows": rows,
            "row_start": _i32(np.zeros(n + 1)), "lens": _i32(np.zeros(n)), "slots": _i32(np.zeros(rows)),
            "positions": _i32(np.zeros(rows)), "free_left": _i32([0])}


def _rope_tables(case):
    """cos / sin of every position's angles, f32, flat: `half` a position."""
    if case["rope"] == "none":
        return None, None
    half = case["dim"] // 2
    n = case["longest"] * (case["heads"] * half if case["rope"] == "row" else half)
    i = torch.arange(n, device=DEV, dtype=torch.float64)
    a = torch.div(i, half, rounding_mode="floor") * 10000.0 ** (-(i % half) / half)
    return a.cos().float(), a.sin().float()


def _prepare_append(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    P, rows, spare, D = case["page"], case["rows"], case["spare_rows"], case["dim"]
    n_pages = -(-rows // P) * 2 + 3
    slots = np.full(rows + spare, -1)
    positions = np.full(rows + spare, -1)
    if rows <= 64:  # decode rows: a page of its own each, anywhere in it
        n_pages = rows + 3
        slots[:rows] = rs.permutation(n_pages)[:rows] * P + rs.randint(0, P, rows)
        positions[:rows] = rs.randint(0, case["longest"], rows)
    else:  # a run of positions over pages in random order
        order, at = rs.permutation(n_pages), int(rs.randint(0, P)) + np.arange(rows)
        slots[:rows] = order[at // P] * P + at % P
        positions[:rows] = at % case["longest"]
    ld = (case["heads"] + 2 * case["kv"]) * D
    cos, sin = _rope_tables(case)
    return {"qkv": torch.randn(rows + spare, ld, generator=_gen(seed, 1), device=DEV), "slots": _i32(slots),
            "positions": _i32(positions), "cos": cos, "sin": sin, "k": _pool(case, n_pages, seed, 2),
            "v": _pool(case, n_pages, seed, 3),
            "q_out": torch.full((rows + spare, case["heads"] * D), 3.0, device=DEV)}


def _attention_lengths(case, seed):
    """(random state, lens, added), as _plan_lengths."""
    rs = np.random.RandomState(case["reqs"])
    lens = _spread(rs, case["reqs"], case["longest"], case["spread"])
    if case["rows"] == 1:
        added = np.ones(case["reqs"], np.int64)
    elif case["rows"] == case["longest"]:
        added = lens
    else:  # half of the requests with one row, the others with a chunk
        added = np.where(rs.rand(case["reqs"]) < 0.5, 1, rs.randint(1, case["rows"] + 1, case["reqs"]))
        added[0] = case["rows"]
        added = np.minimum(added, lens)
    rs = np.random.RandomState(seed % (1 << 32))
    order = rs.permutation(case["reqs"])
    return rs, lens[order], added[order]


def _prepare_attention(case, seed):
    rs, lens, added = _attention_lengths(case, seed)
    pages = -(-lens // case["page"])
    n_pages = int(pages.sum()) + 2
    tables, _ = _tables(rs, pages, n_pages, 1)
    rows = int(added.sum())
    width = case["heads"] * case["dim"]
    return {"q": torch.randn(rows, width, generator=_gen(seed, 1), device=DEV) * 2.0, "tables": _i32(tables),
            "lens": _i32(lens), "row_start": None if case["rows"] == 1 else _i32(np.concatenate([[0], np.cumsum(added)])),
            "k": _pool(case, n_pages, seed, 2), "v": _pool(case, n_pages, seed, 3), "rows": rows,
            "longest": int(lens.max()), "most_added": int(added.max()),
            "out": torch.full((rows, width), 3.0, device=DEV)}


def prepare(case, seed):
    st = {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention}[case["op"]](case, seed)
    st["case"] = case
    return st


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _plain_plan(st):
    P, rows = st["case"]["page"], st["max_rows"]
    cached, added, tables = st["cached"].long(), st["added"].long(), st["tables"]
    lens = cached + added
    row_start = torch.zeros(len(lens) + 1, dtype=torch.long, device=DEV)
    row_start[1:] = added.cumsum(0)
    old, new = (cached + P - 1) // P, (lens + P - 1) // P
    before = (new - old).cumsum(0) - (new - old)
    used = (new - old).sum()
    j = torch.arange(tables.shape[1], device=DEV)[None, :]
    fresh = (j >= old[:, None]) & (j < new[:, None])
    at = st["free_count"].long() - 1 - (before[:, None] + j - old[:, None])
    tables = torch.where(fresh, st["free"][at.clamp(0, len(st["free"]) - 1)], tables)
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(row_start[1:], r, right=True)
    there = b < len(lens)
    b = b.clamp(max=len(lens) - 1)
    p = cached[b] + r - row_start[b]
    slot = tables[b, (p // P).clamp(0, tables.shape[1] - 1)].long() * P + p % P
    return {"tables": tables, "row_start": row_start.int(), "lens": lens.int(),
            "slots": torch.where(there, slot, -1).int(), "positions": torch.where(there, p, -1).int(),
            "free_left": (st["free_count"] - used).int()}


def _rotated(x, positions, cos, sin, half):
    """Pairs (i, i + half) along the last axis of x [rows, ..., 2 half] by the
    angles of the rows' positions."""
    at = positions.long()[:, None] * half + torch.arange(half, device=DEV)
    c, s = cos[at], sin[at]
    if x.dim() == 3:
        c, s = c[:, None], s[:, None]
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1)


def _plain_append(st):
    c = st["case"]
    H, Hk, D, P, rows = c["heads"], c["kv"], c["dim"], c["page"], c["rows"]
    x, p = st["qkv"][:rows], st["positions"][:rows]
    q, k, v = x[:, :H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:]
    if c["rope"] == "row":
        q = _rotated(q, p, st["cos"], st["sin"], H * D // 2)
        k = _rotated(k, p, st["cos"], st["sin"], Hk * D // 2)
    elif c["rope"] == "head":
        q = _rotated(q.view(rows, H, D), p, st["cos"], st["sin"], D // 2).view(rows, -1)
        k = _rotated(k.view(rows, Hk, D), p, st["cos"], st["sin"], D // 2)
    slots = st["slots"][:rows].long()
    page, off = slots // P, slots % P
    st["q_out"][:rows] = q
    st["k"][page, :, off] = k.reshape(rows, Hk, D).to(st["k"].dtype)
    st["v"][page, :, off] = v.reshape(rows, Hk, D).to(st["v"].dtype)
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _gathered(pool, tables, n):
    """The first n keys of every request in f32: [reqs, kv heads, n, head dim]."""
    P = pool.shape[2]
    x = pool[tables[:, :-(-n // P)].long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])[:, :, :n].float()


def _plain_attention(st):
    c = st["case"]
    H, Hk, D = c["heads"], c["kv"], c["dim"]
    G, B, n, most = H // Hk, c["reqs"], st["longest"], st["most_added"]
    k, v = _gathered(st["k"], st["tables"], n), _gathered(st["v"], st["tables"], n)
    lens = st["lens"].long()
    t = torch.arange(n, device=DEV)
    if st["row_start"] is None:
        q = st["q"].view(B, 1, Hk, G, D)
        last = lens[:, None] - 1
    else:
        start = st["row_start"].long()
        added = start[1:] - start[:-1]
        i = torch.arange(most, device=DEV)
        q = st["q"][(start[:-1, None] + i).clamp(max=st["rows"] - 1)].view(B, most, Hk, G, D)
        last = lens[:, None] - added[:, None] + i
    q = q.permute(0, 2, 1, 3, 4).reshape(B, Hk, most * G, D)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    hidden = (t > last[:, :, None]).repeat_interleave(G, 1)[:, None]
    s = s.masked_fill(hidden, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(B, Hk, most, G, D).permute(0, 2, 1, 3, 4).reshape(B * most, H * D)
    if st["row_start"] is not None:
        r = torch.arange(st["rows"], device=DEV)
        b = torch.searchsorted(start[1:], r, right=True)
        o = o[b * most + r - start[b]]
    st["out"].copy_(o)
    return st["out"]


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------
def _own_plan(st):
    from smith_amd import device
    c = st["case"]
    device.check(device.lib.smith_paged_plan(
        device.ops_ctx(), st["cached"].data_ptr(), st["added"].data_ptr(), c["reqs"], st["free"].data_ptr(),
        st["free_count"].data_ptr(), st["n_pages"], c["page"], st["tables"].shape[1], st["max_rows"],
        st["tables"].data_ptr(), st["row_start"].data_ptr(), st["lens"].data_ptr(), st["slots"].data_ptr(),
        st["positions"].data_ptr(), st["free_left"].data_ptr()), "plan")
    return {n: st[n] for n in ("tables", "row_start", "lens", "slots", "positions", "free_left")}


def _own_append(st):
    from smith_amd import device
    c = st["case"]
    cos, sin = st["cos"], st["sin"]
    rows, ld = st["qkv"].shape
    device.check(device.lib.smith_paged_append(
        device.ops_ctx(), TYPES[c["type"]][0], st["qkv"].data_ptr(), ld, rows, st["slots"].data_ptr(),
        st["positions"].data_ptr(), c["heads"], c["kv"], c["dim"], ROPES[c["rope"]],
        cos.data_ptr() if cos is not None else None, sin.data_ptr() if sin is not None else None,
        len(cos) if cos is not None else 0, st["k"].data_ptr(), st["v"].data_ptr(), st["k"].shape[0], c["page"],
        st["q_out"].data_ptr(), st["q_out"].shape[1]), "append")
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _own_attention(st):
    from smith_amd import device
    c = st["case"]
    width = st["q"].shape[1]
    start = st["row_start"]
    device.check(device.lib.smith_paged_attention(
        device.ops_ctx(), TYPES[c["type"]][0], st["q"].data_ptr(), width, st["rows"],
        start.data_ptr() if start is not None else None, st["lens"].data_ptr(), st["tables"].data_ptr(), c["reqs"],
        st["tables"].shape[1], c["heads"], c["kv"], c["dim"], 0.0, st["k"].data_ptr(), st["v"].data_ptr(),
        st["k"].shape[0], c["page"], st["out"].data_ptr(), width), "attention")
    return st["out"]


def run(st):
    if own:
        return {"plan": _own_plan, "append": _own_append, "attention": _own_attention}[st["case"]["op"]](st)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention}[st["case"]["op"]](st)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    if case["op"] == "plan":
        _, cached, added = _plan_lengths(case, 1)
        P, n, rows = case["page"], case["reqs"], int(added.sum())
        pages = int((-(-(cached + added) // P) - -(-cached // P)).sum())
        return {"bytes": 4 * (2 * n + 2 * pages + 2 * n + 1 + 2 * (rows + case["spare_rows"] + 1) + rows // P), "flops": 0}
    H, Hk, D, e = case["heads"], case["kv"], case["dim"], TYPES[case["type"]][2]
    if case["op"] == "append":
        rows = case["rows"]
        angles = {"none": 0, "row": H * D, "head": D}[case["rope"]]
        return {"bytes": rows * (4 * (2 * H + 2 * Hk) * D + 2 * Hk * D * e + 4 * angles + 8),
                "flops": rows * 3 * (H + Hk) * D if angles else 0}
    _, lens, added = _attention_lengths(case, 1)
    keys = (lens * added - added * (added - 1) // 2).sum()
    return {"bytes": int(lens.sum()) * 2 * Hk * D * e + int(added.sum()) * 8 * H * D + 4 * int((-(-lens // case["page"])).sum()),
            "flops": 4.0 * H * D * float(keys)}


# --------------------------------------------------------------------------
# from the definitions in 64 bits, request by request
# --------------------------------------------------------------------------
def _exact_append(case, seed):
    st = _prepare_append(case, seed)
    H, Hk, D, P, rows = case["heads"], case["kv"], case["dim"], case["page"], case["rows"]
    x = st["qkv"].double()[:rows]
    pos = st["positions"][:rows].long()

    def turned(y):  # [rows, n, width]: complex numbers (y_i, y_{i + width / 2}) times e^{i angle}
        half = y.shape[-1] // 2
        at = pos[:, None] * half + torch.arange(half, device=DEV)[None]
        turn = torch.complex(st["cos"].double()[at], st["sin"].double()[at])[:, None]
        z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = x.split([H * D, Hk * D, Hk * D], 1)
    if case["rope"] != "none":
        row = case["rope"] == "row"
        q = turned(q.reshape(rows, 1 if row else H, -1)).reshape(rows, H * D)
        k = turned(k.reshape(rows, 1 if row else Hk, -1)).reshape(rows, Hk * D)
    q_out = st["q_out"].double()
    q_out[:rows] = q
    slots = st["slots"][:rows].long()
    pools = []
    for name, y in (("k", k), ("v", v)):
        flat = st[name].double().transpose(1, 2).reshape(-1, Hk, D)  # slot by slot
        flat[slots] = y.reshape(rows, Hk, D)
        pools.append(flat.view(-1, P, Hk, D).transpose(1, 2).contiguous())
    return {"q": q_out, "k": pools[0], "v": pools[1]}


def _exact_attention(case, seed):
    st = _prepare_attention(case, seed)
    H, Hk, D, P = case["heads"], case["kv"], case["dim"], case["page"]
    lens = st["lens"].tolist()
    start = st["row_start"].tolist() if st["row_start"] is not None else list(range(len(lens) + 1))
    out = torch.empty(st["rows"], H, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        r0, r1 = start[b], start[b + 1]
        if r0 == r1:
            continue
        pages = st["tables"][b, :(n + P - 1) // P].long()
        q = st["q"][r0:r1].double().view(r1 - r0, H, D)
        seen = torch.arange(n, device=DEV)[None, :] <= torch.arange(n - (r1 - r0), n, device=DEV)[:, None]
        for h in range(Hk):
            k = st["k"][pages, h].double().reshape(-1, D)[:n]
            v = st["v"][pages, h].double().reshape(-1, D)[:n]
            for g in range(H // Hk):
                w = torch.where(seen, q[:, h * (H // Hk) + g] @ k.T.contiguous() / D ** 0.5, -math.inf).softmax(1)
                out[r0:r1, h * (H // Hk) + g] = w @ v
    return out.view(st["rows"], H * D)


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers: the plain form's have to be met
    return (_exact_append if case["op"] == "append" else _exact_attention)(case, seed)
