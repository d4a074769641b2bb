"""Pages that requests share: fork and compact against plain forms, alone and in
captured graphs, what they refuse, and what they leave out."""
import ctypes

import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import pages_reference as P_
import paged_reference as R

pytestmark = pytest.mark.gpu


def i32(a):
    return R.upload(np.asarray(a, np.int32))


def last_error():
    return device.lib.smith_last_error(device.ctx()).decode()


def sync_error():
    assert device.lib.smith_sync(device.ctx()) == -1
    return last_error()


def state(seed, n, P, longest, spare=5, share=0.6):
    """lens, tables and the number of pages of requests, some of which share full pages."""
    rs = np.random.RandomState(seed)
    lens = rs.randint(0, longest + 1, n)
    lens[rs.rand(n) < 0.25] //= P
    lens[rs.rand(n) < 0.15] = 0
    whole = rs.rand(n) < 0.2
    lens[whole] = lens[whole] // P * P
    pages = -(-lens // P)
    n_pages = int(pages.sum()) + spare
    order = rs.permutation(n_pages)
    tables = rs.randint(-5, 2 ** 30, (n, int(pages.max()) + 2))  # anything behind a request's pages
    at = 0
    for b in range(n):
        common = 0
        if b and rs.rand() < share:  # as an earlier fork left it
            a = rs.randint(0, b)
            common = rs.randint(0, min(lens[a], lens[b]) // P + 1)
            tables[b, :common] = tables[a, :common]
        tables[b, common:pages[b]] = order[at:at + pages[b] - common]
        at += pages[b] - common
    return rs, lens.astype(np.int32), tables.astype(np.int32), n_pages


def widened(tables):
    """With room for more entries than one workgroup looks through."""
    n, w = tables.shape
    return np.concatenate([tables, np.full((n, max(0, (3 << 14) // n + 1 - w)), 2 ** 30, np.int32)], 1)


def pools_of(rs, count, n_pages, kv, P, D, dtype):
    return [R.stored(rs.standard_normal((n_pages, kv, P, D)).astype(np.float32), dtype) for _ in range(count)]


def moved(pools, copies):
    out = [p.copy() for p in pools]
    for new, old in zip(out, pools):
        for src, dst, keys in copies:
            new[dst, :, :keys] = old[src, :, :keys]
    return out


def parents_of(rs, n, how):
    if how == "same":
        return np.arange(n)
    if how == "one":
        return np.zeros(n, int)
    if how == "none":
        return np.full(n, -1)
    if how == "swap":
        return np.arange(n)[::-1].copy()
    p = rs.randint(-1, n, n)
    return p


@pytest.mark.parametrize("n,P,longest,dtype,kv,D,count", [
    (1, 16, 40, "f16", 2, 16, 1), (2, 1, 7, "f32", 1, 8, 2), (5, 4, 30, "bf16", 3, 24, 4), (24, 16, 200, "f32", 2, 128, 3),
    (64, 8, 100, "f16", 1, 8, 2), (1024, 8, 60, "f16", 1, 8, 1), (1025, 8, 60, "f16", 1, 8, 1), (65, 32, 100, "bf16", 2, 40, 2), (257, 2, 40, "f16", 1, 8, 1), (700, 16, 90, "f32", 1, 8, 1),
    (4096, 16, 33, "f16", 1, 8, 1), (3, 128, 5000, "f16", 8, 128, 2), (2, 16, 9000, "f32", 1, 8, 1)])
@pytest.mark.parametrize("how", ["same", "one", "none", "swap", "any"])
@pytest.mark.parametrize("wide", [False, True])
def test_fork(n, P, longest, dtype, kv, D, count, how, wide):
    rs, lens, tables, n_pages = state(n + P, n, P, longest, 5 + n)
    if wide:
        tables = widened(tables)
    parents = parents_of(rs, n, how).astype(np.int32)
    pools = pools_of(rs, count, n_pages, kv, P, D, dtype)
    marks = np.full(tables.shape, -77, np.int32)
    want = P_.fork(lens, tables, parents, n_pages, P, marks, np.zeros(n_pages, np.int32))
    dev = [R.upload(p, dtype) for p in pools]
    ins = [i32(lens), i32(tables), i32(parents)]
    for _ in range(2):  # the scratch is as it was
        new = S.pagedFork(*ins, dev, newTables=i32(marks))
        device.sync()
        assert np.array_equal(new["lens"].data, want[0])
        assert np.array_equal(new["tables"].data, want[1])
        assert new["freeCount"].data[0] == want[3]
        assert np.array_equal(new["freePages"].data[:want[3]], want[2][:want[3]])
        for got, p in zip(dev, moved(pools, want[4])):
            assert np.array_equal(got.data, p)
    for t, h in zip(ins, (lens, tables, parents)):
        assert np.array_equal(t.data, h)
    for t in dev:
        t.release()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (7, 0), (16, 4), (17, 16), (40, 17), (1000, 3), (2 ** 31, 2 ** 31)])
@pytest.mark.parametrize("P", [1, 4, 16])
@pytest.mark.parametrize("wide", [False, True])
def test_fork_leaves_what_a_window_sees(window, sinks, P, wide):
    rs, lens, tables, n_pages = state(window % 97 + P, 12, P, 120, 20)
    if wide:
        tables = widened(tables)
    pools = pools_of(rs, 2, n_pages, 2, P, 8, "f16")
    # pages that no later row sees were dropped before, too
    for b in range(12):
        for j in range(-(-int(lens[b]) // P)):
            if not P_.kept(j, P, int(lens[b]), window, sinks) and rs.rand() < 0.5:
                tables[b, j] = rs.choice([-1, 2 ** 31 - 1])
    parents = parents_of(rs, 12, "any").astype(np.int32)
    marks = np.full(tables.shape, -77, np.int32)
    want = P_.fork(lens, tables, parents, n_pages, P, marks, np.zeros(n_pages, np.int32), window, sinks)
    dev = [R.upload(p, "f16") for p in pools]
    new = S.pagedFork(i32(lens), i32(tables), i32(parents), dev, window, sinks, i32(marks))
    device.sync()
    assert np.array_equal(new["lens"].data, want[0]) and np.array_equal(new["tables"].data, want[1])
    assert new["freeCount"].data[0] == want[3]
    assert np.array_equal(new["freePages"].data[:want[3]], want[2][:want[3]])
    for got, p in zip(dev, moved(pools, want[4])):
        assert np.array_equal(got.data, p)


@pytest.mark.parametrize("n,P,longest,dtype,kv,D,spare", [
    (1, 16, 40, "f16", 2, 16, 0), (1, 16, 0, "f16", 2, 16, 9), (3, 4, 30, "bf16", 3, 24, 60), (24, 16, 200, "f32", 2, 64, 150),
    (300, 2, 40, "f16", 1, 8, 4000), (1000, 8, 70, "f32", 1, 8, 700), (4096, 16, 33, "f16", 1, 8, 10000)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 3)])
def test_compact(n, P, longest, dtype, kv, D, spare, window, sinks):
    rs, lens, tables, n_pages = state(n + P, n, P, longest, spare)
    pools = pools_of(rs, 2, n_pages, kv, P, D, dtype)
    want = P_.compact(lens, tables, n_pages, P, np.zeros(n_pages, np.int32), window, sinks)
    dev, t = [R.upload(p, dtype) for p in pools], i32(tables)
    new = S.pagedCompact(i32(lens), t, dev, window, sinks)
    device.sync()
    assert np.array_equal(t.data, want[0])
    assert new["freeCount"].data[0] == want[2]
    assert np.array_equal(new["freePages"].data[:want[2]], want[1][:want[2]])
    live = n_pages - want[2]
    for got, p in zip(dev, moved(pools, [(a, b, P) for a, b in want[3]])):
        assert np.array_equal(got.data[:live], p[:live])
    # a compact pool stays as it is
    S.pagedCompact(i32(lens), t, dev, window, sinks)
    device.sync()
    assert np.array_equal(t.data, want[0])
    for x in dev:
        x.release()


@pytest.mark.parametrize("n_pages,n", [(40000, 6), (65536, 30), (65537, 30), (300000, 40), (1 << 20, 3), (1 << 20, 2000)])
def test_large_pools(n_pages, n):
    """Pools whose pages are counted by a launch of their own, and smaller ones."""
    rs = np.random.RandomState(n)
    lens = rs.randint(0, 40, n).astype(np.int32)
    pages = -(-lens // 4)
    tables = np.full((n, 12), -1, np.int32)
    order = rs.permutation(n_pages)[:int(pages.sum())]
    for b, at in enumerate(np.cumsum(pages) - pages):
        tables[b, :pages[b]] = order[at:at + pages[b]]
    parents = rs.randint(-1, n, n).astype(np.int32)
    host = R.stored(rs.standard_normal((n_pages, 1, 4, 8)).astype(np.float32), "f16")
    pool = R.upload(host, "f16")
    want = P_.fork(lens, tables, parents, n_pages, 4, np.zeros_like(tables), np.zeros(n_pages, np.int32))
    new = S.pagedFork(i32(lens), i32(tables), i32(parents), [pool], newTables=S.zeros(tables.shape, "i32"))
    device.sync()
    assert np.array_equal(new["tables"].data, want[1]) and new["freeCount"].data[0] == want[3]
    assert np.array_equal(new["freePages"].data[:want[3]], want[2][:want[3]])
    after = moved([host], want[4])[0]
    assert np.array_equal(pool.data, after)
    c = P_.compact(want[0], want[1], n_pages, 4, np.zeros(n_pages, np.int32))
    got = S.pagedCompact(new["lens"], new["tables"], [pool])
    device.sync()
    assert np.array_equal(new["tables"].data, c[0]) and got["freeCount"].data[0] == c[2]
    live = n_pages - c[2]
    assert np.array_equal(pool.data[:live], moved([after], [(a, b, 4) for a, b in c[3]])[0][:live])
    assert np.array_equal(got["freePages"].data[:c[2]], c[1][:c[2]])
    pool.release()


def test_more_pools_than_one_launch_takes():
    rs, lens, tables, n_pages = state(5, 6, 4, 30, 8)
    pools = pools_of(rs, 900, n_pages, 1, 4, 8, "f16")
    big = R.upload(np.stack(pools).reshape(-1), "f16")
    size = pools[0].nbytes
    pointers = (ctypes.c_void_p * 900)(*[big.buffer + k * size for k in range(900)])
    parents = np.array([1, 1, 1, 0, -1, 5], np.int32)
    want = P_.fork(lens, tables, parents, n_pages, 4, np.zeros_like(tables), np.zeros(n_pages, np.int32))
    ins = [i32(lens), i32(tables), i32(parents)]
    out = [S.zeros([6], "i32"), S.zeros(tables.shape, "i32"), S.zeros([n_pages], "i32"), S.zeros([1], "i32")]
    device.check(device.lib.smith_paged_fork(
        device.ops_ctx(), 1, *[t.buffer for t in ins], 6, tables.shape[1], 0, 0, 1, 8, pointers, 900, n_pages, 4,
        *[t.buffer for t in out]))
    device.sync()
    assert np.array_equal(out[1].data, want[1]) and out[3].data[0] == want[3]
    got = big.data.reshape(900, *pools[0].shape)
    for k, p in enumerate(moved(pools, want[4])):
        assert np.array_equal(got[k], p), k
    # and none
    device.check(device.lib.smith_paged_fork(
        device.ops_ctx(), 1, *[t.buffer for t in ins], 6, tables.shape[1], 0, 0, 1, 8, None, 0, n_pages, 4,
        *[t.buffer for t in out]))
    device.sync()
    assert np.array_equal(out[1].data, want[1]) and out[3].data[0] == want[3]


@pytest.mark.parametrize("wide", [False, True])
def test_a_graph_of_forks_and_compactions(wide):
    """Both captured in one graph, replayed on other requests with eager calls between."""
    ctx = device.ops_ctx()
    P, n = 4, 9
    states = [state(40 + k, n, P, 60, 30) for k in range(5)]
    n_pages = max(s[3] for s in states)
    width = (3 << 14) // n + 1 if wide else max(s[2].shape[1] for s in states)
    rs = np.random.RandomState(1)
    pool = R.upload(pools_of(rs, 1, n_pages, 2, P, 16, "f32")[0], "f32")
    lens, tables, parents = S.zeros([n], "i32"), S.zeros([n, width], "i32"), S.zeros([n], "i32")
    out = [S.zeros([n], "i32"), S.zeros([n, width], "i32"), S.zeros([n_pages], "i32"), S.zeros([1], "i32"),
           S.zeros([n_pages], "i32"), S.zeros([1], "i32")]
    pointers = (ctypes.c_void_p * 1)(pool.buffer)

    def run():
        device.check(device.lib.smith_paged_fork(ctx, 0, lens.buffer, tables.buffer, parents.buffer, n, width, 0, 0, 2, 16,
                                                 pointers, 1, n_pages, P, *[t.buffer for t in out[:4]]))
        device.check(device.lib.smith_paged_compact(ctx, 0, out[0].buffer, out[1].buffer, n, width, 0, 0, 2, 16, pointers,
                                                    1, n_pages, P, out[1].buffer, out[4].buffer, out[5].buffer))

    def load(k):
        _, ln, tb, _ = states[k]
        full = np.zeros((n, width), np.int32)
        full[:, :tb.shape[1]] = tb
        pr = parents_of(np.random.RandomState(k), n, "any").astype(np.int32)
        lens.set_data(ln), tables.set_data(full), parents.set_data(pr)
        out[1].set_data(np.zeros((n, width)))
        old = pool.data
        f = P_.fork(ln, full, pr, n_pages, P, np.zeros_like(full), np.zeros(n_pages, np.int32))
        c = P_.compact(f[0], f[1], n_pages, P, np.zeros(n_pages, np.int32))
        mid = moved([old], f[4])
        return f, c, moved(mid, [(a, b, P) for a, b in c[3]])[0]

    def same(want):
        f, c, host = want
        device.sync()
        assert np.array_equal(out[0].data, f[0]) and np.array_equal(out[1].data, c[0])
        assert np.array_equal(out[2].data[:f[3]], f[2][:f[3]]) and out[3].data[0] == f[3]
        assert np.array_equal(out[4].data[:c[2]], c[1][:c[2]]) and out[5].data[0] == c[2]
        assert np.array_equal(pool.data[:n_pages - c[2]], host[:n_pages - c[2]])

    want = load(0)
    run()
    same(want)
    device.check(device.lib.smith_graph_begin(ctx), "begin")
    run()
    g = device.lib.smith_graph_end(ctx)
    assert g, last_error()
    try:
        for k in (1, 2, 3, 4, 0):
            want = load(k)
            device.check(device.lib.smith_graph_launch(ctx, g))
            same(want)
            want = load((k + 1) % 5)
            run()
            same(want)
        lens.set_data(np.full(n, -1))  # a replay that fails leaves nothing behind
        device.check(device.lib.smith_graph_launch(ctx, g))
        assert "smith_paged_fork" in sync_error()
        want = load(2)
        device.check(device.lib.smith_graph_launch(ctx, g))
        same(want)
    finally:
        device.lib.smith_graph_destroy(g)


@pytest.mark.parametrize("what,message", [
    ("parent", "request 2: its parent"), ("parent_low", "request 2: its parent"), ("negative", "request 1: its length"),
    ("long", "request 1: its length"), ("page", "request 1: a page outside"), ("page_low", "request 1: a page outside"),
    ("free", "more than the 0 pages")])
@pytest.mark.parametrize("call", ["fork", "wide fork", "compact"])
def test_what_does_not_fit_copies_nothing(call, what, message):
    P, n_pages = 4, 7
    lens, parents = np.array([6, 9, 0, 4], np.int32), np.array([1, 0, 1, 3], np.int32)
    tables = np.array([[0, 5, -1], [3, 1, 4], [-1, -1, -1], [2, -1, -1]], np.int32)
    if what == "parent":
        parents[2] = 4
    elif what == "parent_low":
        parents[2] = -2
    elif what == "negative":
        lens[1] = -1
    elif what.startswith("page"):
        tables[1, 1] = 7 if what == "page" else -1
    elif what == "free":
        lens[3], tables[3, 1] = 8, 6
    if call == "compact" and (what.startswith("parent") or what == "free"):
        return  # it has no parents and copies nothing
    if call == "wide fork":
        tables = widened(tables)
    if what == "long":
        lens[1] = tables.shape[1] * P + 1
    rs = np.random.RandomState(0)
    host = pools_of(rs, 1, n_pages, 2, P, 8, "f32")[0]
    pool, t = R.upload(host), i32(tables)
    for _ in range(2):
        if call != "compact":
            new = S.pagedFork(i32(lens), t, i32(parents), [pool])
        else:
            new = S.pagedCompact(i32(lens), t, [pool])
        assert message in sync_error()
        device.sync()  # reported once
        assert np.array_equal(pool.data, host) and np.array_equal(t.data, tables)
        assert new["freeCount"].data[0] == 0
    # and the next call is right
    lens, parents = np.array([6, 9, 0, 4], np.int32), np.array([1, 0, 1, 3], np.int32)
    tables = np.array([[0, 5, -1], [3, 1, 4], [-1, -1, -1], [2, -1, -1]], np.int32)
    want = P_.fork(lens, tables, parents, n_pages, P, np.zeros_like(tables), np.zeros(n_pages, np.int32))
    new = S.pagedFork(i32(lens), i32(tables), i32(parents), [pool], newTables=S.zeros([4, 3], "i32"))
    device.sync()
    assert np.array_equal(new["tables"].data, want[1]) and np.array_equal(pool.data, moved([host], want[4])[0])


def test_pools_beyond_32_bit_offsets():
    """Pools of 5 GiB: copies and moves between their ends."""
    kv, P, D = 4, 64, 64
    n_pages = (5 << 30) // (kv * P * D * 2)
    pools = [S.create([n_pages, kv, P, D], "f16") for _ in range(2)]
    try:
        rs = np.random.RandomState(0)
        page = R.stored(rs.standard_normal((kv, P, D)).astype(np.float32), "f16")
        size = page.nbytes
        src = n_pages - 2
        for t in pools:
            device.upload(t.buffer + src * size, page)
        lens, tables = np.array([P + 30, 0], np.int32), np.array([[n_pages - 1, src], [0, 0]], np.int32)
        new = S.pagedFork(i32(lens), i32(tables), i32([0, 0]), pools)
        device.sync()
        assert new["tables"].data.tolist() == [[n_pages - 1, src], [n_pages - 1, 0]]
        for t in pools:
            got = device.download(t.buffer, size, np.float16).reshape(page.shape)
            assert np.array_equal(got[:, :30], page[:, :30])
        S.pagedCompact(new["lens"], new["tables"], pools)
        device.sync()
        assert new["tables"].data.tolist() == [[2, 1], [2, 0]]
        for t in pools:
            assert np.array_equal(device.download(t.buffer + size, size, np.float16).reshape(page.shape), page)
    finally:
        for t in pools:
            t.release()


# --------------------------------------------------------------------------
# refusals (nothing is launched); addresses are places in one buffer of zeros
# --------------------------------------------------------------------------
_arena = []


def refused(call, **over):
    # two pools of 8 pages x 2 heads x 16 keys x 16 dims of 2 bytes: 8192 bytes
    a = dict(kv=1, lens=4096, tables=4352, parents=4608, n_req=2, max_pages=4, window=0, sinks=0, nKV=2, D=16,
             pools=[1 << 16, 1 << 17], n_pools=2, n_pages=8, P=16, new_lens=8192, new_tables=8448, free=8704, count=8960)
    a.update(over)
    if not _arena:
        _arena.append(S.zeros([1 << 20], "i32"))
    base = _arena[0].buffer
    for k in ("lens", "tables", "parents", "new_lens", "new_tables", "free", "count"):
        a[k] = a[k] if a[k] is None else base + a[k]
    if a["pools"] is not None:
        a["pools"] = (ctypes.c_void_p * max(1, len(a["pools"])))(*[p if p is None else base + p for p in a["pools"]])
    if call == "compact":
        del a["parents"], a["new_lens"]
    rc = getattr(device.lib, "smith_paged_" + call)(device.ops_ctx(), *a.values())
    assert rc == -1
    assert "smith_paged_%s: " % call in last_error()
    return last_error()


@pytest.mark.parametrize("over,message", [
    ({"kv": 3}, "unknown page type 3"), ({"n_req": 0}, "0 requests"), ({"n_req": 4097}, "4097 requests"),
    ({"nKV": 0}, "0 kv heads"), ({"D": 0}, "head_dim 0"), ({"D": 12}, "head_dim 12"), ({"D": 136}, "head_dim 136"),
    ({"P": 0}, "page size 0"), ({"P": 24}, "page size 24"), ({"n_pages": 0}, "pool of 0 pages"),
    ({"n_pages": 1 << 27}, "pool of"), ({"max_pages": 0}, "block tables of 0"), ({"max_pages": 1 << 27}, "block tables of"),
    ({"sinks": 4}, "4 sinks without a window"), ({"lens": None}, "null buffer"), ({"tables": None}, "null buffer"),
    ({"new_tables": None}, "null buffer"), ({"free": None}, "null buffer"), ({"count": None}, "null buffer"),
    ({"pools": None}, "pools (up to"), ({"n_pools": 4097}, "4097 pools"), ({"pools": [1 << 16, None]}, "page pools"),
    ({"pools": [1 << 16, (1 << 17) + 8]}, "16-byte aligned"), ({"pools": [1 << 17, (1 << 17) - 8176]}, "two pools overlap"),
    ({"pools": [1 << 16, 1 << 16]}, "two pools overlap"), ({"pools": [4096, 1 << 17]}, "a pool overlaps an input"),
    ({"pools": [8448 - 8192 + 16, 1 << 17], "lens": 1 << 18, "tables": (1 << 18) + 64, "parents": (1 << 18) + 256}, "a pool overlaps an output"),
    ({"new_tables": 4352 + 4}, "an output overlaps an input"), ({"free": 4096}, "an output overlaps an input"),
    ({"count": 8704}, "two outputs overlap"), ({"free": 8448}, "two outputs overlap")])
@pytest.mark.parametrize("call", ["fork", "compact"])
def test_refusals(call, over, message):
    assert message in refused(call, **over)


@pytest.mark.parametrize("over,message", [
    ({"parents": None}, "null buffer"), ({"new_lens": None}, "null buffer"), ({"new_lens": 4096}, "an output overlaps an input"),
    ({"new_tables": 4352}, "an output overlaps an input"), ({"new_lens": 8448}, "two outputs overlap")])
def test_fork_refusals(over, message):
    assert message in refused("fork", **over)


def test_a_free_list_that_is_too_short():
    lens, t, pool = i32([3]), i32([[0]]), S.zeros([9, 1, 4, 8], "f16")
    short = S.zeros([8], "i32")
    pointers = (ctypes.c_void_p * 1)(pool.buffer)
    out = [S.zeros([1], "i32") for _ in range(3)]
    assert device.lib.smith_paged_fork(device.ops_ctx(), 1, lens.buffer, t.buffer, i32([0]).buffer, 1, 1, 0, 0, 1, 8, pointers,
                                       1, 9, 4, out[0].buffer, out[1].buffer, short.buffer, out[2].buffer) == -1
    assert "room for 8 of 9 pages" in last_error()
    with pytest.raises(ValueError, match="pagedFork: parents"):
        S.pagedFork(lens, t, i32([0, 1]), [pool])
    with pytest.raises(ValueError, match="pagedFork: pools"):
        S.pagedFork(lens, t, i32([0]), [pool, S.zeros([9, 1, 4, 8], "f32")])
    with pytest.raises(ValueError, match="pools are"):
        S.pagedCompact(lens, t, [])
    for call, args in ((S.pagedFork, (lens, t, i32([0]), [pool])), (S.pagedCompact, (lens, t, [pool]))):
        for window, sinks in ((-1, 0), (0, 1), (3, -1)):
            with pytest.raises(ValueError, match="a window of %d keys and %d sinks" % (window, sinks)):
                call(*args, window, sinks)


def test_a_window_longer_than_any_request():
    """More than fits 32 bits is no window of 0."""
    rs, lens, tables, n_pages = state(3, 5, 4, 40, 3)
    pool = R.upload(pools_of(rs, 1, n_pages, 1, 4, 8, "f16")[0], "f16")
    got = [S.pagedFork(i32(lens), i32(tables), i32(np.arange(5)), [pool], window, sinks, i32(tables))
           for window, sinks in ((0, 0), (2 ** 32 + 1, 2 ** 32))]
    device.sync()
    for name in ("lens", "tables", "freeCount"):
        assert np.array_equal(got[0][name].data, got[1][name].data)
