"""Paged KV cache: several requests share one pool of pages per layer.

The reference's cache is one request's, [kvHeads, maxSeqLen, headDim] per layer
(gguf_cache.js:14-28).  Here a layer's keys and values are pools of pages,
[pages, kvHeads, pageSize, headDim], and a block table per request names its
pages in order, so that requests of any lengths take only the pages that they
fill.  A step of any mix of prompts, chunks and decode rows is

    pagedPlan       block tables, slots and positions from the lengths
    pagedAppend     rotary positions, then k and v into their slots   (per layer)
    pagedAttention  the rows' attention over the pages                (per layer)

on Tensors (one call into libsmith.so each, include/smith.h states what each
reads and writes).  PagedCache keeps the pools, tables and lengths of a model's
requests on the device; forwardPagedStep of a loaded GGUF model runs on it.
"""
import numpy as np

from . import device
from . import tensor as T

KV_TYPES = {"f32": 0, "f16": 1, "bf16": 2}
ROPE_NONE, ROPE_ROW, ROPE_HEAD = 0, 1, 2
MAX_REQUESTS = 4096  # of one step


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


def pagedAttention(q, lens, tables, kPages, vPages, rowStart=None, scale=0.0, out=None):
    """Causal attention of rows q [rows, numHeads * headDim] over the pages
    (smith_paged_attention): request b's rows are rowStart[b] .. rowStart[b+1]-1,
    or row b alone without rowStart.  Returns out (a new tensor if None is given,
    whose rows behind the last one are then undefined)."""
    nPages, nKV, P, hd = _pools(kPages, vPages, "pagedAttention")
    rows, width = q.shape
    n = lens.shape[0]
    if q.dtype != "f32" or width % hd:
        raise ValueError("pagedAttention: q is f32 [rows, heads * %d], got %s %s" % (hd, q.dtype, q.shape))
    _want(lens, [n], "i32", "pagedAttention: lens")
    _want(tables, [n, tables.shape[-1]], "i32", "pagedAttention: tables")
    if rowStart is not None:
        _want(rowStart, [n + 1], "i32", "pagedAttention: rowStart")
    if out is None:
        out = T.create([rows, width])
    _want(out, [rows, width], "f32", "pagedAttention: out")
    device.check(device.lib.smith_paged_attention(
        device.ops_ctx(), KV_TYPES[kPages.dtype], q.buffer, width, rows,
        rowStart.buffer if rowStart is not None else None, lens.buffer, tables.buffer, n, tables.shape[1], width // hd,
        nKV, hd, scale, kPages.buffer, vPages.buffer, nPages, P, out.buffer, width), "pagedAttention")
    return out


def _release(tensors):
    for t in tensors:
        t.release()


class PagedCache:
    """The paged cache of a model's requests: per layer the pools k and v, and on
    the device the block tables [requests, maxPages], lengths and free list, which
    the host mirrors in `lens` and `freeCount`.  A request is its number, 0 ..
    requests - 1; it takes pages as it grows and gives them back with release()."""

    def __init__(self, config, requests, pages, pageSize=16, dtype="f16"):
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
        self.maxPages = -(-config["maxSeqLen"] // pageSize)
        self.lens = np.zeros(requests, np.int32)
        self.freeCount = pages
        self.layers, self._rows, self._turn, self._tensors = [], None, 0, []
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
        return {"rowStart": self._row_start, "lens": self._lens[b], "slots": slots, "positions": positions,
                "tables": self._tables}

    def state(self):
        """For restore()."""
        return self._turn, self.lens, self.freeCount

    def restore(self, state):
        """Back to a state() from before the last plan(), if nothing was released
        since: what that step read on the device is still there."""
        self._turn, self.lens, self.freeCount = state

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
        device.check(device.lib.smith_paged_attention(
            device.ops_ctx(), KV_TYPES[self.dtype], q, ld, rows, plan["rowStart"].buffer, plan["lens"].buffer,
            plan["tables"].buffer, self.requests, self.maxPages, numHeads, k.shape[1], k.shape[3], 0.0, k.buffer,
            v.buffer, self.pages, self.pageSize, out, numHeads * k.shape[3]), "paged attention")

    def release(self, request):
        """The request's pages back to the free list; its number is free for another."""
        self._there()
        if not 0 <= request < self.requests:
            raise ValueError("paged cache: request %d of %d" % (request, self.requests))
        n = -(-int(self.lens[request]) // self.pageSize)
        if not n:
            return
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


def createPagedCache(config, requests, pages, pageSize=16, dtype="f16"):
    """A PagedCache for a model of this config (GGUFModel.config's fields of
    createGGUFCache): pools of `pages` pages of pageSize keys per layer."""
    return PagedCache(config, requests, pages, pageSize, dtype)
