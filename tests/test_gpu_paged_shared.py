"""Attention of groups of requests that have their first keys in common, against 64 bits."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import pages_reference as P_
import paged_reference as R
from test_gpu_paged import i32, last_error, placed, room_for_many, sync_error

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


# keys that the block tables have room for, so that the shared keys are computed apart: 48 MB and more
def wide(tables, nKV, D, dtype, P):
    keys = (48 << 20) // (2 * nKV * D * (4 if dtype == "f32" else 2)) // len(tables)
    more = max(0, keys // P + 1 - tables.shape[1])
    return np.concatenate([tables, np.full((len(tables), more), 2 ** 31 - 1, np.int32)], 1)


def case(seed, dtype, H, nKV, D, P, widths, shared, own, added, q_std=2.0, apart=True):
    """Groups of widths[g] requests, the first shared[g] keys of each the same (a
    partly filled page a copy), own[b] keys behind them, the last added[b] of rows."""
    rs = np.random.RandomState(seed)
    start = np.concatenate([[0], np.cumsum(widths)])
    n = int(start[-1])
    of = np.repeat(np.arange(len(widths)), widths)
    shared, own, added = (np.broadcast_to(np.asarray(x), m).astype(np.int64) for x, m in ((shared, len(widths)), (own, n), (added, n)))
    lens = (shared[of] + own).astype(np.int32)
    pages = -(-lens // P)
    n_pages = int(pages.sum()) + 2
    order = rs.permutation(n_pages)
    tables = rs.randint(-2 ** 31, 2 ** 31 - 1, (n, int(pages.max()) + 1)).astype(np.int32)
    at = 0
    k, v = (R.stored(rs.standard_normal((n_pages, nKV, P, D)), dtype) for _ in range(2))
    for b in range(n):
        first, full = start[of[b]], shared[of[b]] // P
        if b == first:
            full = 0
        else:
            tables[b, :full] = tables[first, :full]
        tables[b, full:pages[b]] = order[at:at + pages[b] - full]
        at += pages[b] - full
        part = shared[of[b]] % P
        if b != first and part:
            for pool in (k, v):
                pool[tables[b, full], :, :part] = pool[tables[first, full], :, :part]
    if apart:
        tables = wide(tables, nKV, D, dtype, P)
    q = (rs.standard_normal((int(added.sum()), H, D)) * q_std).astype(np.float32)
    row_start = np.concatenate([[0], np.cumsum(added)]).astype(np.int32)
    return q, row_start, lens, tables, k, v, start.astype(np.int32), shared.astype(np.int32)


def run(q, row_start, lens, tables, k, v, start, shared, ragged, room=0, scale=0.0):
    rows, W = len(q), q.shape[1] * q.shape[2]
    room = max(room, rows)
    hq = np.full((room, W), np.nan, np.float32)
    hq[:rows] = q.reshape(rows, -1)
    out = R.upload(np.full((room, W), 5, np.float32))
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start) if ragged else None,
                     scale, out, groupStart=i32(start), shared=i32(shared))
    device.sync()
    assert (out.data[rows:] == 5).all()
    return out.data[:rows]


def everything(b, at, t):
    return t >= 0


def check(got, c, dtype, scale=None, seen=everything):
    q, row_start, lens, tables, k, v = c[:6]
    P_.check_attention(got, P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype),
                                         seen, scale), q.shape[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shared", [0, 1, 7, 15, 16, 17, 31, 64, 65, 100, 128, 300, 1000])
@pytest.mark.parametrize("P", [4, 16, 64])
@pytest.mark.parametrize("apart", [True, False])
def test_one_group(dtype, shared, P, apart):
    own = np.array([1, 2, 16, 33, 60])
    c = case(shared + P, dtype, 4, 2, 32, P, [5], shared, own, 1, apart=apart)
    check(run(*c, False), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,nKV,D,P", [(1, 1, 8, 1), (9, 3, 64, 8), (10, 2, 80, 32), (12, 4, 96, 16), (20, 1, 128, 128), (33, 1, 40, 2)])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("apart", [True, False])
def test_heads_pages_and_groups(dtype, H, nKV, D, P, ragged, apart):
    """Groups of one and of many requests, with and without shared keys, requests that sit out."""
    rs = np.random.RandomState(H)
    widths = [1, 7, 2, 1, 12]
    own = rs.randint(4, 50, 23)
    added = rs.randint(0, 5, 23) if ragged else 1
    c = case(H + D, dtype, H, nKV, D, P, widths, [40, 133, 0, 0, 70], own, added, apart=apart)
    check(run(*c, ragged), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P", [8, 16])
@pytest.mark.parametrize("room", [0, room_for_many(8, 2, 6)])
def test_chunks_behind_a_shared_prompt(dtype, P, room):
    """Rows of chunks, by both kernels for the own keys."""
    c = case(P, dtype, 8, 2, 40, P, [4, 2], [333, 90], [70, 40, 5, 33, 100, 65], [70, 13, 1, 0, 100, 30])
    check(run(*c, True, room), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,shared", [(2, 9000), (40, 3000), (200, 700)])
def test_long_shared_keys_are_cut(dtype, width, shared):
    rs = np.random.RandomState(width)
    c = case(width, dtype, 8, 2, 64, 16, [width], shared, rs.randint(1, 40, width), 1)
    check(run(*c, False), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_own_keys_are_cut(dtype):
    c = case(9, dtype, 8, 2, 64, 16, [3], 500, [3000, 20, 900], 1)
    check(run(*c, False), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,groups", [(70, 70), (300, 3), (4096, 64), (4096, 4096)])
def test_many_requests(dtype, n, groups):
    rs = np.random.RandomState(n)
    cut = np.sort(rs.choice(np.arange(1, n), groups - 1, replace=False))
    widths = np.diff(np.concatenate([[0], cut, [n]]))
    c = case(n, dtype, 2, 1, 16, 8, widths, rs.randint(0, 40, groups), rs.randint(1, 20, n), 1)
    check(run(*c, False), c, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,groups", [(4096, 4096), (4096, 3), (4000, 200)])
def test_most_requests_with_many_columns(dtype, n, groups):
    """By the kernels of many columns where their tables fit beside the stages."""
    rs = np.random.RandomState(groups)
    widths = np.full(groups, n // groups)
    widths[:n % groups] += 1
    c = case(n + groups, dtype, 8, 1, 8, 8, widths, rs.randint(0, 20, groups), rs.randint(4, 9, n), 4)
    check(run(*c, True), c, dtype)


@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 4)])
@pytest.mark.parametrize("starts", [[0, 5, 3, 8, 9], [0, 3, 9, 4, 6], [3, 1, 9, 4, 9], [9, 0, 9, 0, 9], [0, 9, 9, 2, 2], [-1, 4, 5, 7, 9]])
@pytest.mark.parametrize("apart", [True, False])
def test_row_start_out_of_order_stays_inside(starts, room, apart):
    """Starts that go back and forth: no request reads what its group did not leave, and
    the calls after it are right."""
    c = q, row_start, lens, tables, k, v, start, shared = case(6, "f16", 4, 2, 32, 16, [2, 2], [40, 30], [20, 20, 20, 20],
                                                               [3, 2, 2, 2], apart=apart)
    rows = max(room, len(q))
    hq = np.zeros((rows, 128), np.float32)
    hq[:len(q)] = q.reshape(len(q), -1)
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(starts), 0.0, None,
                     groupStart=i32(start), shared=i32(shared))
    assert "smith_paged_attention" in sync_error()
    device.sync()
    check(run(*c, True, room), c, "f16")


@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 9)])
@pytest.mark.parametrize("starts", [[0, 3, -1, 9], [0, 6, 2, 9], [0, 9, 0, 9], [4, 9, 9, 9], [0, -5, 2 ** 31 - 1, 9]])
@pytest.mark.parametrize("apart", [True, False])
def test_groups_that_leave_out_or_repeat_requests_stay_inside(starts, room, apart):
    """Requests of no group, and of two, behind a call whose shared keys were cut."""
    c = q, row_start, lens, tables, k, v, start, shared = case(8, "f16", 4, 2, 32, 16, [2, 5, 2], [900, 40, 30], 20,
                                                               [3, 2, 2, 2, 1, 0, 4, 5, 1], apart=apart)
    check(run(*c, True, room), c, "f16")
    rows = max(room, len(q))
    hq = np.zeros((rows, 128), np.float32)
    hq[:len(q)] = q.reshape(len(q), -1)
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start), 0.0, None,
                     groupStart=i32(starts), shared=i32([30, 40, 30]))
    assert "smith_paged_attention_shared: group" in sync_error()
    device.sync()
    check(run(*c, True, room), c, "f16")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("ragged", [False, True])
def test_dominating_keys_and_far_scores(dtype, where, ragged):
    """All of the weight on one side of the join, and scores of any size."""
    for size in (1.0, 30.0):
        c = case(4, dtype, 4, 2, 64, 16, [4], 100, [30, 20, 9, 33], 2 if ragged else 1)
        q, _, lens, tables, k, v = c[:6]
        q *= np.float32(size)
        for b in range(4):
            t = 50 if where == "shared" else lens[b] - 3
            head = q[2 * b if ragged else b].reshape(2, 2, 64).mean(1)
            k[tables[b, t // 16], :, t % 16] = R.stored((head * np.float32(2 / size)).astype(np.float32), dtype)
        check(run(*c, ragged), c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("junk", [np.nan, np.inf])
@pytest.mark.parametrize("ragged,room", [(False, 0), (True, 0), (True, room_for_many(6, 2, 4))])
def test_what_is_not_finite(dtype, junk, ragged, room):
    """Behind the shared and the own keys, and before the own ones in a request's own
    copy of the page, nobody sees it; in a shared key all of the group do, in a key of
    its own its request's later rows."""
    c = case(6, dtype, 6, 2, 24, 16, [3, 1], [37, 20], [30, 9, 40, 25], [5, 1, 20, 3] if ragged else 1)
    q, row_start, lens, tables, k, v, start, shared = c
    clean = [k.copy(), v.copy()]
    bad = {"f32": np.float32(junk), "f16": np.float16(junk),
           "bf16": np.uint16(np.float32(junk).view(np.uint32) >> 16 | (0x40 if np.isnan(junk) else 0))}[dtype]
    used = np.zeros((k.shape[0], 16), bool)
    for b, n in enumerate(lens):
        t = np.arange(n)
        if b in (1, 2):
            t = t[t >= 37]
        used[tables[b, t // 16], t % 16] = True
    for pool in (k, v):
        pool.transpose(0, 2, 1, 3)[~used] = bad
    want = P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(clean[0], dtype), R.value(clean[1], dtype), everything)
    got = run(*c, ragged, room)
    P_.check_attention(got, want, 24)
    # a row's own key
    b, t = 2, lens[2] - (10 if ragged else 1)
    keep = v[tables[b, t // 16], :, t % 16, 3].copy()
    v[tables[b, t // 16], :, t % 16, 3] = bad
    got = run(*c, ragged, room).reshape(q.shape)
    spoiled = np.arange(row_start[3] - (10 if ragged else 1), row_start[3])
    assert not np.isfinite(got[spoiled][..., 3]).any()
    rest = np.delete(np.arange(len(q)), spoiled)
    P_.check_attention(got[rest], [x[rest] for x in want], 24)
    v[tables[b, t // 16], :, t % 16, 3] = keep
    # a shared one
    v[tables[0, 1], :, 5, 3] = bad
    got = run(*c, ragged, room).reshape(q.shape)
    n = row_start[3] if ragged else 3
    assert not np.isfinite(got[:n][..., 3]).any()
    P_.check_attention(got[n:], [x[n:] for x in want], 24)


@pytest.mark.parametrize("ragged", [False, True])
def test_strides_and_rows_behind_the_last(ragged):
    c = q, row_start, lens, tables, k, v, start, shared = case(8, "bf16", 6, 3, 56, 16, [2, 3], [40, 70], 20, 3 if ragged else 1)
    H, D, rows, W = 6, 56, len(q), 6 * 56
    room = rows + 9 if ragged else rows
    ld_q, ld_o = W + 3, W + 5
    hq = np.random.RandomState(1).standard_normal(1 + room * ld_q).astype(np.float32)
    ho = np.random.RandomState(2).standard_normal(3 + room * ld_o).astype(np.float32)
    for r in range(rows):
        hq[1 + r * ld_q:1 + r * ld_q + W] = q[r].ravel()
    tq, to, tk, tv = R.upload(hq), R.upload(ho), R.upload(k), R.upload(v)
    rs, ln, tb, gs, sh = i32(row_start), i32(lens), i32(tables), i32(start), i32(shared)
    assert device.lib.smith_paged_attention_shared(
        device.ops_ctx(), 2, tq.buffer + 4, ld_q, room, rs.buffer if ragged else None, ln.buffer, tb.buffer, 5, tables.shape[1],
        gs.buffer, sh.buffer, 2, H, 3, D, 0.0, tk.buffer, tv.buffer, k.shape[0], 16, to.buffer + 12, ld_o) == 0, last_error()
    device.sync()
    got = to.data
    at = [slice(3 + r * ld_o, 3 + r * ld_o + W) for r in range(rows)]
    check(np.stack([got[s] for s in at]), c, "bf16")
    for s in at:
        got[s] = ho[s]
    assert np.array_equal(got, ho)


@pytest.mark.parametrize("bad,message,lost", [
    ("short", "request 1: more shared keys", [1]), ("negative", "group 0: ", [0, 1, 2]), ("long", "group 0: ", [0, 1, 2]),
    ("start", "group 0: ", [0, 1, 2, 3, 4]), ("order", "group ", [0, 1, 2, 3, 4]), ("end", "group 1: ", [3, 4]), ("len", "request 4: its length", [4]),
    ("page", "request 0: a page outside", [0, 1, 2])])
@pytest.mark.parametrize("apart", [True, False])
def test_leaves_out_what_does_not_fit(bad, message, lost, apart):
    c = q, row_start, lens, tables, k, v, start, shared = case(5, "f16", 4, 2, 32, 16, [3, 2], [40, 20], [5, 6, 7, 8, 9], 1,
                                                               apart=apart)
    lens, start, shared, now = lens.copy(), start.copy(), shared.copy(), tables.copy()
    if bad == "short":
        lens[1] = 40
    elif bad == "negative":
        shared[0] = -1
    elif bad == "long":
        shared[0] = tables.shape[1] * 16 + 1
    elif bad == "start":
        start[0] = 1
    elif bad == "order":
        start[1] = 6
    elif bad == "end":
        start[2] = 4
    elif bad == "len":
        lens[4] = -1
    else:
        now[0, 1] = k.shape[0]
        if not apart:
            message = "a page outside"
    out = R.upload(np.full((5, 128), 5, np.float32))
    S.pagedAttention(R.upload(q.reshape(5, -1)), i32(lens), i32(now), R.upload(k), R.upload(v), None, 0.0, out,
                     groupStart=i32(start), shared=i32(shared))
    assert message in sync_error()
    device.sync()
    got = out.data
    if bad == "len":
        assert (got[lost] == 5).all()
    rest = [b for b in range(5) if b not in lost]
    want = P_.attention(q.astype(np.float64), row_start, c[2], tables, R.value(k, "f16"), R.value(v, "f16"), everything)
    P_.check_attention(got[rest], [x[rest] for x in want], 32)
    check(run(*c, False), c, "f16")  # and the call after it


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_graphs_on_one_scratch(dtype):
    """Captured steps of two caches, replayed in turn while the requests grow, beside eager calls."""
    ctx, steps = device.ops_ctx(), []
    for seed, (widths, shared, n, ragged) in enumerate([([20], 600, 1, False), ([2, 3], [90, 40], 7, True)]):
        c = q, row_start, lens, tables, k, v, start, sh = case(seed, dtype, 8, 2, 32, 16, widths, shared, 40, n)
        ln, gs, sd = i32(lens), i32(start), i32(sh)
        out = S.create([len(q), 256])
        args = (R.upload(q.reshape(len(q), -1)), ln, i32(tables), R.upload(k), R.upload(v), i32(row_start) if ragged else None,
                0.0, out, 0, 0, gs, sd)
        S.pagedAttention(*args)
        steps.append([c, ln, sd, args, None])
    device.sync()
    try:
        for st in steps:
            device.check(device.lib.smith_graph_begin(ctx), "begin")
            S.pagedAttention(*st[3])
            st[4] = device.lib.smith_graph_end(ctx)
            assert st[4], last_error()
        for turn in range(4):
            lengths = []
            for (q, row_start, lens, tables, k, v, start, sh), ln, sd, args, g in steps:
                now = lens - 3 * turn
                ln.set_data(now)
                sd.set_data(sh - 5 * turn)
                lengths.append(now)
                args[7].set_data(np.zeros(args[7].shape, np.float32))
            for st in steps:
                device.check(device.lib.smith_graph_launch(ctx, st[4]))
            for st, now in zip(steps, lengths):
                got = st[3][7].data
                check(got, (*st[0][:2], now, *st[0][3:]), dtype)
            S.pagedAttention(*steps[turn % 2][3][:7], None, 0, 0, *steps[turn % 2][3][10:])
            device.sync()
    finally:
        for st in steps:
            if st[4]:
                device.lib.smith_graph_destroy(st[4])


@pytest.mark.parametrize("over,message", [
    ({"kv": 3}, "unknown page type 3"), ({"H": 5}, "5 heads not a multiple of 2"), ({"D": 12}, "head_dim 12"),
    ({"max_pages": 0}, "block tables of 0"), ({"n_req": 4097, "max_rows": 4097}, "4097 requests"),
    ({"max_rows": 3}, "max_rows 3 for one row"), ({"ld_q": 63}, "row strides 63"), ({"k": None}, "page pools"),
    ({"lens": None}, "null buffer"), ({"groups": None}, "null buffer"), ({"shared": None}, "null buffer"),
    ({"n_groups": 0}, "0 groups of 2"), ({"n_groups": 3}, "3 groups of 2"), ({"out": 4096 + 256}, "out overlaps q"),
    ({"groups": 1 << 20}, "out overlaps an input"), ({"shared": (1 << 20) + 8}, "out overlaps an input")])
def test_refusals(over, message):
    a = dict(kv=1, q=4096, ld_q=64, max_rows=2, row_start=None, lens=4096, tables=4096, n_req=2, max_pages=4, groups=8192,
             shared=8448, n_groups=1, H=4, nKV=2, D=16, scale=0.0, k=4096, v=4096, n_pages=8, P=16, out=1 << 20, ld_out=64)
    a.update(over)
    assert device.lib.smith_paged_attention_shared(
        device.ops_ctx(), *placed(a, "q", "row_start", "lens", "tables", "groups", "shared", "k", "v", "out")) == -1
    assert "smith_paged_attention_shared: " in last_error() and message in last_error()


def test_wrapper_refusals():
    k = S.zeros([2, 1, 16, 8], "f16")
    args = (S.zeros([2, 8]), S.zeros([2], "i32"), S.zeros([2, 1], "i32"), k, k)
    g, s = S.zeros([2], "i32"), S.zeros([1], "i32")
    for more, message in (({"groupStart": g}, "take groupStart and shared"), ({"shared": s}, "take groupStart and shared"),
                          ({"groupStart": g, "shared": s, "window": 3}, "no window"), ({"groupStart": s, "shared": s}, "groupStart: i32"),
                          ({"window": -1}, "a window of -1")):
        with pytest.raises(ValueError, match=message):
            S.pagedAttention(*args, **more)
