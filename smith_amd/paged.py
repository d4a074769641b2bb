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
    added: [n] i32; freePages [..] and freeCount [1] i32: the free list; tables
    [n, maxPages] i32, new pages are entered.  Returns {rowStart [n + 1], lens
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
    if rope and (cos is None or sin is None or cos.size != sin.size):
        raise ValueError("pagedAppend: rotary positions need tables cos and sin of one size")
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
