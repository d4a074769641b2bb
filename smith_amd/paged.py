"""Paged KV cache: several requests share one pool of pages per layer.

The reference's cache is one request's, [kvHeads, maxSeqLen, headDim] per layer
(gguf_cache.js:14-28).  Here a layer's keys and values are pools of pages,
[pages, kvHeads, pageSize, headDim], and a block table per request names its
pages in order, so that requests of any lengths take only the pages that they
fill.  A step of any mix of prompts, chunks and decode rows is

    pagedPlan       block tables, slots and positions from the lengths
    pagedAppend     rotary positions, then k and v into their slots   (per layer)
    pagedAttention  the rows' attention over the pages                (per layer)

and between steps

    pagedFork       requests go on from others, whose full pages they share
    pagedCompact    the live pages at the pools' low end

on Tensors (one call into libsmith.so each, include/smith.h states what each
reads and writes).  PagedCache keeps the pools, tables and lengths of a model's
requests on the device; forwardPagedStep of a loaded GGUF model runs on it.
"""
import collections
import ctypes
import itertools

import numpy as np

from . import device
from . import tensor as T

KV_TYPES = {"f32": 0, "f16": 1, "bf16": 2}
ROPE_NONE, ROPE_ROW, ROPE_HEAD = 0, 1, 2
MAX_REQUESTS = 4096  # of one step
MOST_KEYS = 2 ** 31 - 1  # of a request


def _window(window, sinks, what):
    """Both as they fit the calls: no request is longer."""
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError("%s: a window of %d keys and %d sinks" % (what, window, sinks))
    return min(window, MOST_KEYS), min(sinks, MOST_KEYS)


def _want(t, shape, dtype, what):
    if list(t.shape) != list(shape) or t.dtype != dtype:
        raise ValueError("%s: %s %s wanted, got %s %s" % (what, dtype, list(shape), t.dtype, list(t.shape)))


def _pools(kPages, vPages, what):
    if kPages.dtype not in KV_TYPES or len(kPages.shape) != 4:
        raise ValueError("%s: pages are [pages, kvHeads, pageSize, headDim] of f32, f16 or bf16" % what)
    _want(vPages, kPages.shape, kPages.dtype, what + ": vPages")
    return kPages.shape


def pagedPlan(cached, added, freePages, freeCount, tables, nPages, pageSize, maxRows):
    """Block tables, slots and positions of a step (smith_paged_plan).  cached,
    added: [n] i32; freePages [..] and freeCount [1] i32: the free list, its first
    freeCount entries; tables [n, maxPages] i32, new pages are entered.  Returns {rowStart [n + 1], lens
    [n], slots [maxRows], positions [maxRows], freeLeft [1]}, all i32."""
    n = cached.shape[0]
    _want(cached, [n], "i32", "pagedPlan: cached")
    _want(added, [n], "i32", "pagedPlan: added")
    _want(freeCount, [1], "i32", "pagedPlan: freeCount")
    _want(freePages, freePages.shape[:1], "i32", "pagedPlan: freePages")
    _want(tables, [n, tables.shape[-1]], "i32", "pagedPlan: tables")
    plan = {"rowStart": T.create([n + 1], "i32"), "lens": T.create([n], "i32"), "slots": T.create([maxRows], "i32"),
            "positions": T.create([maxRows], "i32"), "freeLeft": T.create([1], "i32")}
    device.check(device.lib.smith_paged_plan(
        device.ops_ctx(), cached.buffer, added.buffer, n, freePages.buffer, freeCount.buffer, nPages, pageSize,
        tables.shape[1], maxRows, tables.buffer, plan["rowStart"].buffer, plan["lens"].buffer, plan["slots"].buffer,
        plan["positions"].buffer, plan["freeLeft"].buffer), "pagedPlan")
    return plan


def pagedAppend(qkv, slots, positions, numHeads, kPages, vPages, rope=ROPE_NONE, cos=None, sin=None):
    """Rows [q | k | v] into the pages; returns the rotated q [rows, numHeads *
    headDim] (smith_paged_append)."""
    nPages, nKV, P, hd = _pools(kPages, vPages, "pagedAppend")
    rows, ld = qkv.shape
    _want(qkv, [rows, (numHeads + 2 * nKV) * hd], "f32", "pagedAppend: qkv")
    _want(slots, [rows], "i32", "pagedAppend: slots")
    _want(positions, [rows], "i32", "pagedAppend: positions")
    if rope and (cos is None or sin is None or cos.size != sin.size or (cos.dtype, sin.dtype) != ("f32", "f32")):
        raise ValueError("pagedAppend: rotary positions need tables cos and sin, f32 of one size")
    q = T.create([rows, numHeads * hd])
    device.check(device.lib.smith_paged_append(
        device.ops_ctx(), KV_TYPES[kPages.dtype], qkv.buffer, ld, rows, slots.buffer, positions.buffer, numHeads, nKV,
        hd, rope, cos.buffer if rope else None, sin.buffer if rope else None, cos.size if rope else 0, kPages.buffer,
        vPages.buffer, nPages, P, q.buffer, numHeads * hd), "pagedAppend")
    return q


def pagedAttention(q, lens, tables, kPages, vPages, rowStart=None, scale=0.0, out=None, window=0, sinks=0,
                   groupStart=None, shared=None):
    """Causal attention of rows q [rows, numHeads * headDim] over the pages
    (smith_paged_attention): request b's rows are rowStart[b] .. rowStart[b+1]-1,
    or row b alone without rowStart.  Returns out (a new tensor if None is given,
    whose rows behind the last one are then undefined).

    window > 0: a row sees the last `window` keys up to its own and the first
    `sinks` (smith_paged_attention_window).  groupStart [n + 1], shared [n] i32: the
    requests groupStart[g] .. groupStart[g+1]-1 have their first shared[g] keys in
    common, which are read once for all of them (smith_paged_attention_shared)."""
    nPages, nKV, P, hd = _pools(kPages, vPages, "pagedAttention")
    rows, width = q.shape
    n = lens.shape[0]
    if q.dtype != "f32" or width % hd:
        raise ValueError("pagedAttention: q is f32 [rows, heads * %d], got %s %s" % (hd, q.dtype, q.shape))
    _want(lens, [n], "i32", "pagedAttention: lens")
    _want(tables, [n, tables.shape[-1]], "i32", "pagedAttention: tables")
    if rowStart is not None:
        _want(rowStart, [n + 1], "i32", "pagedAttention: rowStart")
    window, sinks = _window(window, sinks, "pagedAttention")
    name, reach = "smith_paged_attention", ()
    if groupStart is not None or shared is not None:
        if groupStart is None or shared is None or window:
            raise ValueError("pagedAttention: shared keys take groupStart and shared, and no window")
        groups = shared.shape[0]
        _want(shared, [groups], "i32", "pagedAttention: shared")
        _want(groupStart, [groups + 1], "i32", "pagedAttention: groupStart")
        name, reach = "smith_paged_attention_shared", (groupStart.buffer, shared.buffer, groups)
    elif window:
        name, reach = "smith_paged_attention_window", (window, sinks)
    if out is None:
        out = T.create([rows, width])
    _want(out, [rows, width], "f32", "pagedAttention: out")
    device.check(getattr(device.lib, name)(
        device.ops_ctx(), KV_TYPES[kPages.dtype], q.buffer, width, rows,
        rowStart.buffer if rowStart is not None else None, lens.buffer, tables.buffer, n, tables.shape[1], *reach,
        width // hd, nKV, hd, scale, kPages.buffer, vPages.buffer, nPages, P, out.buffer, width), "pagedAttention")
    return out


def _all_pools(pools, what):
    """(shape, dtype, host array of the addresses) of pools that are alike."""
    pools = list(pools)
    if not pools or pools[0].dtype not in KV_TYPES or len(pools[0].shape) != 4:
        raise ValueError("%s: pools are [pages, kvHeads, pageSize, headDim] of f32, f16 or bf16" % what)
    for t in pools:
        _want(t, pools[0].shape, pools[0].dtype, what + ": pools")
    return pools[0].shape, pools[0].dtype, (ctypes.c_void_p * len(pools))(*[t.buffer for t in pools])


def pagedFork(lens, tables, parents, pools, window=0, sinks=0, newTables=None):
    """Request b goes on from request parents[b] (itself, another, -1: none) as it
    was, sharing its full pages; a partly filled page stays with the first and is
    copied for the others in all `pools` (smith_paged_fork).  lens, parents [n] and
    tables [n, maxPages] i32.  Returns {lens [n], tables, freePages [pages],
    freeCount [1]}, i32; newTables is the tensor that tables are written to."""
    n = lens.shape[0]
    _want(lens, [n], "i32", "pagedFork: lens")
    _want(parents, [n], "i32", "pagedFork: parents")
    _want(tables, [n, tables.shape[-1]], "i32", "pagedFork: tables")
    window, sinks = _window(window, sinks, "pagedFork")
    shape, dtype, pointers = _all_pools(pools, "pagedFork")
    if newTables is None:
        newTables = T.create(tables.shape, "i32")
    _want(newTables, tables.shape, "i32", "pagedFork: newTables")
    new = {"lens": T.create([n], "i32"), "tables": newTables, "freePages": T.create([shape[0]], "i32"),
           "freeCount": T.create([1], "i32")}
    device.check(device.lib.smith_paged_fork(
        device.ops_ctx(), KV_TYPES[dtype], lens.buffer, tables.buffer, parents.buffer, n, tables.shape[1], window, sinks,
        shape[1], shape[3], pointers, len(pointers), shape[0], shape[2], new["lens"].buffer, newTables.buffer,
        new["freePages"].buffer, new["freeCount"].buffer), "pagedFork")
    return new


def pagedCompact(lens, tables, pools, window=0, sinks=0):
    """The live pages moved to the pools' low end, in all `pools`; `tables` name
    them there (smith_paged_compact).  Returns {freePages [pages], freeCount [1]}."""
    n = lens.shape[0]
    _want(lens, [n], "i32", "pagedCompact: lens")
    _want(tables, [n, tables.shape[-1]], "i32", "pagedCompact: tables")
    window, sinks = _window(window, sinks, "pagedCompact")
    shape, dtype, pointers = _all_pools(pools, "pagedCompact")
    new = {"freePages": T.create([shape[0]], "i32"), "freeCount": T.create([1], "i32")}
    device.check(device.lib.smith_paged_compact(
        device.ops_ctx(), KV_TYPES[dtype], lens.buffer, tables.buffer, n, tables.shape[1], window, sinks, shape[1],
        shape[3], pointers, len(pointers), shape[0], shape[2], tables.buffer, new["freePages"].buffer,
        new["freeCount"].buffer), "pagedCompact")
    return new


def _release(tensors):
    for t in tensors:
        t.release()


# Keys and values of a layer's shared keys that are read once instead of once a
# request, in bytes, from which the launch that computes them apart is worth its time
# (6 us a layer, in which the card reads 30 MB).
SHARED_BYTES = 32 << 20


class PagedCache:
    """The paged cache of a model's requests: per layer the pools k and v, and on
    the device the block tables [requests, maxPages], lengths and free list, which
    the host mirrors in `lens` and `freeCount`.  A request is its number, 0 ..
    requests - 1; it takes pages as it grows and gives them back with release().
    fork() lets requests go on from others on shared pages.  With a window a row
    sees the last `window` keys up to its own and the first `sinks`, and pages that no
    later row sees are given back when others are needed, or by trim()."""

    def __init__(self, config, requests, pages, pageSize=16, dtype="f16", window=0, sinks=0):
        if dtype not in KV_TYPES:
            raise ValueError("createPagedCache: pages of %s (f32, f16 or bf16)" % dtype)
        if not 1 <= requests <= MAX_REQUESTS:
            raise ValueError("createPagedCache: %d requests (1 .. %d)" % (requests, MAX_REQUESTS))
        if pageSize < 1 or pageSize & (pageSize - 1):
            raise ValueError("createPagedCache: page size %d is no power of two" % pageSize)
        if pages < 1 or pages * pageSize >= 1 << 31:
            raise ValueError("createPagedCache: %d pages of %d keys" % (pages, pageSize))
        if config["headDim"] % 8 or not 8 <= config["headDim"] <= 128:
            raise ValueError("createPagedCache: heads of %d dims (8, 16 .. 128)" % config["headDim"])
        self.requests, self.pages, self.pageSize, self.dtype = requests, pages, pageSize, dtype
        self.window, self.sinks = _window(window, sinks, "createPagedCache")
        self.maxPages = -(-config["maxSeqLen"] // pageSize)
        self.lens = np.zeros(requests, np.int32)
        self.freeCount = pages
        self.layers, self._rows, self._turn, self._tensors = [], None, 0, []
        # from the first fork on: of each request a number for each of its pages (None: given
        # back), and how many requests name it; what they share, host and device
        self._ids, self._named, self._next_id = None, collections.Counter(), 0
        self._groups, self._group_tensors, self._spare = [], None, None
        self._read_twice = 0  # bytes of a layer's shared keys and values, once for each further request
        try:
            self._allocate(config)
        except BaseException:
            self.free()
            raise

    def _allocate(self, config):
        def hold(t):
            self._tensors.append(t)
            return t
        n, shape = self.requests, [self.pages, config["numKVHeads"], self.pageSize, config["headDim"]]
        for _ in range(config["numLayers"]):
            self.layers.append({name: hold(T.create(shape, self.dtype)) for name in ("k", "v")})
        self._tables = hold(T.zeros([n, self.maxPages], "i32"))
        self._free = hold(T.tensor(np.arange(self.pages - 1, -1, -1), dtype="i32"))  # page 0 goes first
        # what a step reads and what it writes, in turn
        self._lens = [hold(T.zeros([n], "i32")) for _ in range(2)]
        self._count = [hold(T.tensor([self.pages], dtype="i32")) for _ in range(2)]
        self._added = hold(T.zeros([n], "i32"))
        self._row_start = hold(T.zeros([n + 1], "i32"))

    def check_model(self, config):
        """Raises ValueError unless the pools are those of a model of this config."""
        k = self.layers[0]["k"].shape if self.layers else [0] * 4
        if (len(self.layers), k[1], k[3]) != (config["numLayers"], config["numKVHeads"], config["headDim"]):
            raise ValueError("paged step: a cache of %d layers of %d heads of %d, a model of %d of %d of %d" % (
                len(self.layers), k[1], k[3], config["numLayers"], config["numKVHeads"], config["headDim"]))

    def _there(self):
        if not self._tensors:
            raise ValueError("paged cache: it was freed")

    def _pages(self, n):
        return -(-int(n) // self.pageSize)

    def make_room(self, added):
        """Gives back what the window has passed, if the rows `added` need it."""
        if not self.window:
            return
        lens = self.lens.astype(np.int64)
        if int((-(-(lens + added) // self.pageSize) - -(-lens // self.pageSize)).sum()) > self.freeCount:
            self.trim()

    def plan(self, added):
        """The step in which request b brings added[b] rows: {rowStart, lens, slots,
        positions, tables}.  Nothing happens (ValueError) if it does not fit."""
        self._there()
        added = np.asarray(added, np.int64)
        rows = int(added.sum())
        lens = self.lens + added
        if added.shape != (self.requests,) or (added < 0).any() or not rows:
            raise ValueError("paged step: the rows of %d requests, one at least" % self.requests)
        if (lens > self.maxPages * self.pageSize).any():
            raise ValueError("paged step: request %d grows past %d keys" % (int(lens.argmax()), self.maxPages * self.pageSize))
        new = int((-(-lens // self.pageSize) - -(-self.lens // self.pageSize)).sum())
        if new > self.freeCount:
            raise ValueError("paged step: %d new pages, %d are free" % (new, self.freeCount))
        if self._rows is None or self._rows["slots"].shape[0] < rows:
            # rows behind a step's last stay at slot -1: one pair of buffers serves all sizes up to theirs
            room, pair = max(256, rows), {}
            try:
                for name in ("slots", "positions"):
                    pair[name] = T.create([room], "i32")
            except BaseException:
                _release(pair.values())
                raise
            _release((self._rows or {}).values())
            self._rows = pair
        self._added.set_data(added)
        a, b = self._turn, 1 - self._turn
        slots, positions = self._rows["slots"], self._rows["positions"]
        device.check(device.lib.smith_paged_plan(
            device.ops_ctx(), self._lens[a].buffer, self._added.buffer, self.requests, self._free.buffer,
            self._count[a].buffer, self.pages, self.pageSize, self.maxPages, slots.shape[0], self._tables.buffer,
            self._row_start.buffer, self._lens[b].buffer, slots.buffer, positions.buffer, self._count[b].buffer),
            "paged step")
        self._turn, self.lens, self.freeCount = b, lens.astype(np.int32), self.freeCount - new
        if self._ids is not None:
            for r in np.nonzero(added)[0]:
                self._name(r)
        return {"rowStart": self._row_start, "lens": self._lens[b], "slots": slots, "positions": positions,
                "tables": self._tables}

    def _name(self, r):
        """Numbers for the pages that request r has and had not."""
        ids = self._ids[r]
        while len(ids) < self._pages(self.lens[r]):
            ids.append(self._next_id)
            self._named[self._next_id] = 1
            self._next_id += 1

    def state(self):
        """For restore()."""
        return self._turn, self.lens, self.freeCount

    def restore(self, state):
        """Back to a state() from before the last plan(), if nothing was released
        since: what that step read on the device is still there."""
        self._turn, self.lens, self.freeCount = state
        if self._ids is not None:
            for ids, n in zip(self._ids, self.lens):
                while len(ids) > self._pages(n):
                    del self._named[ids.pop()]

    # --- requests that go on from others ---
    def _kept(self, j, n):
        """Whether page j of a request of n keys has a sink or one that a later row sees."""
        P = self.pageSize
        return not self.window or j * P < self.sinks or (j + 1) * P + self.window > n + 1

    def _seen(self, ids, n):
        """A copy of a request's numbers of pages, None for those that its window has passed."""
        return [x if self._kept(j, int(n)) else None for j, x in enumerate(ids)] if self.window else ids.copy()

    @staticmethod
    def _count_names(ids):
        named = collections.Counter(itertools.chain.from_iterable(ids))
        named.pop(None, None)
        return named

    def fork(self, parents):
        """Request b goes on from request parents[b] as it was: itself, another, or -1,
        none.  Full pages are shared; a partly filled one stays with the first request
        that goes on from its own, and is copied for the others.  Nothing happens
        (ValueError) if there are too few pages for the copies."""
        self._there()
        parents = np.asarray(parents)
        if parents.shape != (self.requests,) or parents.dtype.kind not in "iu" or not (
                (parents >= -1) & (parents < self.requests)).all():
            raise ValueError("paged fork: parents are %d numbers of requests or -1" % self.requests)
        if self._ids is None:
            self._ids = [[] for _ in range(self.requests)]
            for r in range(self.requests):
                self._name(r)
        ids, seen, next_id = [], set(), self._next_id
        lens = np.where(parents >= 0, self.lens[parents], 0).astype(np.int32)
        for p, n in zip(parents, lens):
            mine = self._seen(self._ids[p], n) if p >= 0 else []
            if p in seen and n % self.pageSize:
                mine[-1], next_id = next_id, next_id + 1
            seen.add(p)
            ids.append(mine)
        named = self._count_names(ids)
        if len(named) > self.pages:
            raise ValueError("paged fork: %d pages, there are %d" % (len(named), self.pages))
        tables, free, todo = self._spares()
        a, b = self._turn, 1 - self._turn
        todo.set_data(parents)
        pools = [layer[name].buffer for layer in self.layers for name in ("k", "v")]
        shape = self.layers[0]["k"].shape if self.layers else [0, 1, 0, 8]
        device.check(device.lib.smith_paged_fork(
            device.ops_ctx(), KV_TYPES[self.dtype], self._lens[a].buffer, self._tables.buffer, todo.buffer, self.requests,
            self.maxPages, self.window, self.sinks, shape[1], shape[3], (ctypes.c_void_p * len(pools))(*pools), len(pools),
            self.pages, self.pageSize, self._lens[b].buffer, tables.buffer, free.buffer, self._count[b].buffer), "paged fork")
        self._turn, self.lens, self.freeCount = b, lens, self.pages - len(named)
        self._spare = (self._tables, self._free, todo)
        self._tables, self._free = tables, free
        self._ids, self._named, self._next_id = ids, named, next_id
        self._find_groups()

    def _spares(self):
        """Tables, a free list and parents for a fork to write and read (and what
        _find_groups writes): there before it begins."""
        if self._spare is None:
            got, n = [], self.requests
            try:
                for shape in ([n, self.maxPages], [self.pages], [n], [n + 1], [n]):
                    got.append(T.create(shape, "i32"))
            except BaseException:
                _release(got)
                raise
            self._tensors += got
            self._spare, self._group_tensors = tuple(got[:3]), tuple(got[3:])
        return self._spare

    def _find_groups(self):
        """Runs of requests whose first pages are the same ones: [first, behind the last,
        pages], a request that shares none by itself."""
        groups = []
        for r, ids in enumerate(() if self.window else self._ids):
            if groups:
                first, _, most = groups[-1]
                same, of = 0, self._ids[first]
                if most and ids[:most] == of[:most]:
                    same = most
                else:
                    while same < min(len(ids), len(of)) and ids[same] == of[same]:
                        same += 1
                # (a run is not cut to less than half of what it shares for one more)
                if same and (r == first + 1 or same * 2 > most):
                    groups[-1] = [first, r + 1, min(most, same) if most else same]
                    continue
            groups.append([r, r + 1, 0])
        self._groups, self._read_twice = [], 0
        if self.window or len(groups) == self.requests:
            return
        start, shared = np.full(self.requests + 1, self.requests), np.zeros(self.requests, np.int64)
        start[:len(groups)] = [g[0] for g in groups]
        shared[:len(groups)] = [g[2] * self.pageSize for g in groups]
        self._group_tensors[0].set_data(start)
        self._group_tensors[1].set_data(shared)
        self._groups = groups
        k = self.layers[0]["k"] if self.layers else None
        size = 2 * k.shape[1] * k.shape[3] * (4 if self.dtype == "f32" else 2) if k else 0
        self._read_twice = size * sum((b - a - 1) * n * self.pageSize for a, b, n in groups)

    def trim(self):
        """Gives back the pages that the window has passed."""
        self.fork(np.arange(self.requests))

    def compact(self):
        """Moves the pages that requests have to the pools' low end; their number."""
        self._there()
        tables, free, _ = self._spares()
        a, b = self._turn, 1 - self._turn
        pools = [layer[name].buffer for layer in self.layers for name in ("k", "v")]
        shape = self.layers[0]["k"].shape if self.layers else [0, 1, 0, 8]
        device.check(device.lib.smith_paged_compact(
            device.ops_ctx(), KV_TYPES[self.dtype], self._lens[a].buffer, self._tables.buffer, self.requests, self.maxPages,
            self.window if self._ids is not None else 0, self.sinks if self._ids is not None else 0, shape[1], shape[3],
            (ctypes.c_void_p * len(pools))(*pools), len(pools), self.pages, self.pageSize, tables.buffer, free.buffer,
            self._count[b].buffer), "paged compact")
        # the lengths are those of this turn: only the count is new
        device.check(device.lib.smith_copy_d2d(device.ops_ctx(), self._count[a].buffer, 0, self._count[b].buffer, 0, 4),
                     "paged compact")
        self._spare = (self._tables, self._free, self._spare[2])
        self._tables, self._free = tables, free
        if self._ids is not None and self.window:  # pages that the window had passed are free now
            self._ids = [self._seen(ids, n) for ids, n in zip(self._ids, self.lens)]
            self._named = self._count_names(self._ids)
            self.freeCount = self.pages - len(self._named)
        return self.pages - self.freeCount

    def resize(self, pages):
        """Pools of `pages` pages, as many as the requests have at least (compact() says how
        many that is); the device holds the old and the new ones for a while."""
        live = self.compact()
        if pages < max(1, live) or pages * self.pageSize >= 1 << 31:
            raise ValueError("paged cache: %d pages for the %d that its requests have" % (pages, live))
        got = []
        try:
            for layer in self.layers:
                for name in ("k", "v"):
                    got.append(T.create([pages] + layer[name].shape[1:], self.dtype))
            got.append(T.tensor(np.arange(pages - 1, -1, -1), dtype="i32"))
            got.append(T.create([pages], "i32"))
            ctx = device.ops_ctx()
            for old, new in zip([layer[name] for layer in self.layers for name in ("k", "v")], got):
                if live:
                    device.check(device.lib.smith_copy_d2d(ctx, new.buffer, 0, old.buffer, 0, old.nbytes // self.pages * live),
                                 "paged cache")
            device.sync()  # the old pools are read until here
            device.check(device.lib.smith_set_i32(ctx, self._count[self._turn].buffer, pages - live), "paged cache")
        except BaseException:
            _release(got)
            raise
        spare_tables, _, todo = self._spare
        gone = [layer.pop(name) for layer in self.layers for name in ("k", "v")] + [self._free, self._spare[1]]
        for layer in self.layers:
            layer["k"], layer["v"] = got.pop(0), got.pop(0)
        self._free, spare_free = got
        self._spare = (spare_tables, spare_free, todo)
        drop = {id(t) for t in gone}
        self._tensors = [t for t in self._tensors if id(t) not in drop]
        self._tensors += [layer[name] for layer in self.layers for name in ("k", "v")] + got
        _release(gone)
        self.pages, self.freeCount = pages, pages - live

    def append(self, layer, plan, qkv, ld, rows, numHeads, rope, cos, sin, ropeLen):
        """A layer's rows [q | k | v] (device pointer, row stride ld floats) into its
        pages; q is rotated in place."""
        self._there()
        k, v = self.layers[layer]["k"], self.layers[layer]["v"]
        device.check(device.lib.smith_paged_append(
            device.ops_ctx(), KV_TYPES[self.dtype], qkv, ld, rows, plan["slots"].buffer, plan["positions"].buffer,
            numHeads, k.shape[1], k.shape[3], rope, cos, sin, ropeLen, k.buffer, v.buffer, self.pages, self.pageSize,
            qkv, ld), "paged append")

    def attention(self, layer, plan, q, ld, rows, numHeads, out):
        """A layer's attention of the step's rows into out [rows, numHeads * headDim]."""
        self._there()
        k, v = self.layers[layer]["k"], self.layers[layer]["v"]
        name, reach = "smith_paged_attention", ()
        if self.window:
            name, reach = "smith_paged_attention_window", (self.window, self.sinks)
        elif self._groups and self._read_twice >= SHARED_BYTES:
            name = "smith_paged_attention_shared"
            reach = (*(t.buffer for t in self._group_tensors), len(self._groups))
        device.check(getattr(device.lib, name)(
            device.ops_ctx(), KV_TYPES[self.dtype], q, ld, rows, plan["rowStart"].buffer, plan["lens"].buffer,
            plan["tables"].buffer, self.requests, self.maxPages, *reach, numHeads, k.shape[1], k.shape[3], 0.0, k.buffer,
            v.buffer, self.pages, self.pageSize, out, numHeads * k.shape[3]), "paged attention")

    def release(self, request):
        """The request's pages back to the free list, but for those that others share;
        its number is free for another."""
        self._there()
        if not 0 <= request < self.requests:
            raise ValueError("paged cache: request %d of %d" % (request, self.requests))
        n = self._pages(self.lens[request])
        if not n:
            return
        if self._ids is not None:
            if any(x is None or self._named[x] > 1 for x in self._ids[request]):
                parents = np.arange(self.requests)
                parents[request] = -1
                return self.fork(parents)
            for x in self._ids[request]:
                del self._named[x]
            self._ids[request] = []
            self._find_groups()
        ctx, a = device.ops_ctx(), self._turn
        device.check(device.lib.smith_copy_d2d(ctx, self._free.buffer, 4 * self.freeCount, self._tables.buffer,
                                               4 * request * self.maxPages, 4 * n), "paged cache")
        device.check(device.lib.smith_set_i32(ctx, self._lens[a].buffer + 4 * request, 0), "paged cache")
        device.check(device.lib.smith_set_i32(ctx, self._count[a].buffer, self.freeCount + n), "paged cache")
        self.freeCount += n
        self.lens[request] = 0

    def free(self):
        """Gives the device memory back; the cache is not used after it."""
        _release(self._tensors + list((self._rows or {}).values()))
        self.layers, self._rows, self._tensors = [], None, []
        self._spare = self._group_tensors = None


def createPagedCache(config, requests, pages, pageSize=16, dtype="f16", window=0, sinks=0):
    """A PagedCache for a model of this config (GGUFModel.config's fields of
    createGGUFCache): pools of `pages` pages of pageSize keys per layer, whose rows
    see all keys, or the last `window` and the first `sinks`."""
    return PagedCache(config, requests, pages, pageSize, dtype, window, sinks)
