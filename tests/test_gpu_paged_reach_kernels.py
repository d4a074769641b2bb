"""Every kernel of attention over part of the keys (a window; shared keys and a request's
own), by name, against 64 bits.  Which one runs depends on max_rows and the visible keys:
rows behind the last one, which nobody reads or writes, make room for the kernels of many
rows."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import accuracy_reference as A
import pages_reference as P_
import paged_reference as R
from test_gpu_paged import attention_case, i32, last_error, room_for_many, sync_error
from test_gpu_paged_shared import case as shared_case, everything
from test_gpu_paged_window import drop, visible

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


def held(D):
    return 64 if D <= 64 else 96 if D <= 96 else 128


def room_for_window(dtype, H, nKV, n_req, seen):
    """max_rows with which a window's rows are answered by the kernel of many rows."""
    return max(-(-((64 if dtype == "f32" else 8) << 20) // (H * seen)), 24 * n_req * nKV // H + 1)


def ran(name):
    """Whether the kernel of this name did, of the launches recorded; they are forgotten."""
    if not name.endswith("_s"):
        device.profile_read(name + "_s")
    return device.profile_read(name)[1] > 0


def attend(q, row_start, lens, tables, k, v, kernels, room=0, ragged=True, **reach):
    """pagedAttention with max_rows = room by the kernels of these names."""
    rows, W = len(q), q.shape[1] * q.shape[2]
    room = max(room, rows)
    tail = min(room, rows + 64)
    made = [S.create([room, W]) for _ in range(2)]
    try:
        hq, ho = np.full((tail, W), np.nan, np.float32), np.full((tail, W), 5, np.float32)
        hq[:rows] = q.reshape(rows, W)
        for t, host in zip(made, (hq, ho)):
            device.upload(t.buffer, host)
        ins = [i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start)]
        more = {name: i32(x) if name in ("groupStart", "shared") else x for name, x in reach.items()}
        made += ins + [t for t in more.values() if isinstance(t, S.Tensor)]
        device.profile_read("")
        device.profile_kernels(True)
        try:
            S.pagedAttention(made[0], *ins[:4], ins[4] if ragged else None, 0.0, made[1], **more)
        finally:
            device.profile_kernels(False)
        for name in kernels:
            assert ran("smith_paged_attention" + name), name
        device.profile_read("")
        device.sync()
        got = device.download(made[1].buffer, tail * W * 4, np.float32).reshape(tail, W)
        assert (got[rows:] == 5).all()
        return got[:rows].reshape(q.shape)
    finally:
        for t in made:
            t.release()


def check(got, want, D, q_std=None):
    P_.check_attention(got, want, D)
    if q_std:
        A.check_norm(got, want[0], want[3], q_std)


# --------------------------------------------------------------------------
# a window
# --------------------------------------------------------------------------
def window(seed, dtype, H, nKV, D, P, lens, added, win, sinks, kind, q_std=2.0, bar=False):
    q, row_start, ln, tables, k, v = attention_case(seed, dtype, H, nKV, D, P, lens, added, q_std)
    tables = drop(seed, tables, ln, added, P, win, sinks, k.shape[0])
    name = "_window_%s%s_d%d%s" % ("rows_" if kind == "rows" else "", dtype, held(D), "_s" if kind == "small" else "")
    seen = min(win + sinks, tables.shape[1] * P)
    got = attend(q, row_start, ln, tables, k, v, [name], room_for_window(dtype, H, nKV, len(lens), seen) if kind == "rows" else 0,
                 kind == "rows" or any(a != 1 for a in added), window=win, sinks=sinks)
    want = P_.attention(q.astype(np.float64), row_start, ln, tables, R.value(k, dtype), R.value(v, dtype), visible(win, sinks))
    check(got, want, D, q_std if bar else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("kind", ["few", "small", "rows"])
@pytest.mark.parametrize("q_std", list(A.BARS))
def test_window_accuracy(dtype, D, kind, q_std):
    lens = [1, 17, 64, 100, 129, 400, 700, 1500]
    added = [1, 5, 33, 20, 1, 40, 0, 17] if kind == "rows" else [1] * 8
    window(D, dtype, 4, 2, D, 4 if kind == "small" else 16, lens, added, 300, 20, kind, q_std, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("win,sinks,H,nKV,D,P", [
    (5, 3, 6, 2, 24, 8), (16, 0, 9, 3, 64, 16), (40, 17, 6, 2, 80, 16), (64, 100, 12, 4, 96, 32), (90, 1, 6, 2, 128, 8),
    (333, 20, 20, 1, 104, 128), (5000, 4, 6, 2, 72, 16), (33, 33, 33, 1, 40, 64),
    (50, 9, 70, 1, 32, 16)])
def test_window_rows(dtype, win, sinks, H, nKV, D, P):
    window(win + P, dtype, H, nKV, D, P, [150, 30, 64, 400, 9], [80, 1, 20, 70, 0], win, sinks, "rows")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,nKV,D", [(16, 4, 64), (16, 4, 96), (32, 8, 128)])
def test_window_rows_cut_and_joined(dtype, H, nKV, D):
    window(D, dtype, H, nKV, D, 32, [3000], [40], 1500, 40, "rows")


@pytest.mark.parametrize("dtype", TYPES)
def test_window_rows_of_most_requests(dtype):
    rs = np.random.RandomState(2)
    window(5, dtype, 8, 1, 8, 8, rs.randint(4, 40, 4096), [4] * 4096, 300, 2, "rows")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [40, 96, 128])
@pytest.mark.parametrize("junk", [np.nan, np.inf])
def test_window_rows_ignore_what_they_do_not_see(dtype, D, junk):
    """What is not finite between the sinks and the window, in dropped pages and behind a
    request; and in a key that only some rows of a block see."""
    lens, added = [150, 40, 64, 300], [2, 20, 64, 1]
    H, nKV, P, win, sinks = 6, 2, 16, 23, 5
    q, row_start, ln, tables, k, v = attention_case(3, dtype, H, nKV, D, P, lens, added)
    clean = [k.copy(), v.copy()]
    bad = {"f32": np.float32(junk), "f16": np.float16(junk),
           "bf16": np.uint16(np.float32(junk).view(np.uint32) >> 16 | (0x40 if np.isnan(junk) else 0))}[dtype]
    used = np.zeros((k.shape[0], P), bool)
    for b, n in enumerate(lens):
        t = np.arange(n)
        t = t[(t > n - added[b] - win) | (t < sinks)]
        used[tables[b, t // P], t % P] = True
    for pool in (k, v):
        pool.transpose(0, 2, 1, 3)[~used] = bad
    spoiled = []
    for b, t in ((1, 30), (2, 20)):
        for pool in (k, v):
            pool[tables[b, t // P], :, t % P, 3] = bad
        first = ln[b] - added[b]
        spoiled += [row_start[b] + i for i in range(added[b]) if t <= first + i < t + win]
    got = attend(q, row_start, ln, drop(3, tables, ln, added, P, win, sinks, k.shape[0]), k, v,
                 ["_window_rows_%s_d%d" % (dtype, held(D))], room_for_window(dtype, H, nKV, 4, win + sinks), window=win, sinks=sinks)
    assert not np.isfinite(got[spoiled][..., 3]).any()
    want = P_.attention(q.astype(np.float64), row_start, ln, tables, R.value(clean[0], dtype), R.value(clean[1], dtype),
                        visible(win, sinks))
    rest = np.delete(np.arange(len(q)), spoiled)
    assert np.isfinite(got[rest]).all()
    check(got[rest], [x[rest] for x in want], D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128])
def test_a_window_of_everything_by_rows_is_plain_attention(dtype, D):
    c = q, row_start, lens, tables, k, v = attention_case(8, dtype, 4, 2, D, 16, [400, 33, 90], [50, 33, 1])
    a = attend(*c, ["_rows_%s_d%d" % (dtype, held(D))], room_for_many(4, 2, 3))
    b = attend(*c, ["_window_rows_%s_d%d" % (dtype, held(D))], room_for_window(dtype, 4, 2, 3, 400), window=400)
    # two sums of the same products: each off by less than the bar of 64 bits
    assert np.linalg.norm(a - b) <= 2 * A.BARS[2.0] * np.linalg.norm(a)


@pytest.mark.parametrize("dtype", TYPES)
def test_window_rows_a_page_outside_the_pool(dtype):
    q, row_start, lens, tables, k, v = attention_case(5, dtype, 4, 2, 32, 16, [140, 30], [1, 1])
    tables[0, 7] = k.shape[0]  # in its window
    room = room_for_window(dtype, 4, 2, 2, 52)
    made = [S.create([room, 128]) for _ in range(2)]
    device.upload(made[0].buffer, q.reshape(2, -1))
    made += [i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start)]
    S.pagedAttention(made[0], *made[2:6], made[6], 0.0, made[1], 50, 2)
    assert "request 0: a page outside" in sync_error()
    device.sync()
    for t in made:
        t.release()


@pytest.mark.parametrize("D", [64, 128])
def test_window_rows_of_pages_beyond_32_bit_offsets(D):
    H, nKV, P = 8, 4, 64
    n_pages = (5 << 30) // (nKV * P * D * 2)
    q, row_start, lens, tables, k, v = attention_case(17, "f16", H, nKV, D, P, [700, 130], [1, 70], spare=0)
    used = -(-lens // P)
    far = tables.copy()
    for b in range(2):
        tables[b, used[b]:] = 0
        far[b, :used[b]] = n_pages - 1 - tables[b, :used[b]]
    room = room_for_window("f16", H, nKV, 2, 108)
    made = [S.create([n_pages, nKV, P, D], "f16") for _ in range(2)] + [S.create([room, H * D]) for _ in range(2)]
    try:
        for t, host in zip(made, (k, v)):
            for i in range(len(host)):
                device.upload(t.buffer + (n_pages - 1 - i) * host[i].nbytes, np.ascontiguousarray(host[i]))
        device.upload(made[2].buffer, q.reshape(len(q), -1))
        device.profile_read("")
        device.profile_kernels(True)
        try:
            S.pagedAttention(made[2], i32(lens), i32(far), *made[:2], i32(row_start), 0.0, made[3], 99, 9)
        finally:
            device.profile_kernels(False)
        assert ran("smith_paged_attention_window_rows_f16_d%d" % held(D))
        device.sync()
        got = device.download(made[3].buffer, q.nbytes, np.float32)
        check(got, P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, "f16"), R.value(v, "f16"),
                                visible(99, 9)), D)
    finally:
        for t in made:
            t.release()


# --------------------------------------------------------------------------
# shared keys and a request's own
# --------------------------------------------------------------------------
def shared_names(kind, dtype, D, apart):
    of = {"few": ("", ""), "small": ("", ""), "wide": ("rows_", ""), "chunks": ("rows_", "rows_")}[kind]
    tail = "%s_d%d%s" % (dtype, held(D), "_s" if kind == "small" else "")
    return (["_shared_%s%s" % (of[0], tail)] if apart else []) + ["_own_%s%s" % (of[1], tail)]


def shared(seed, dtype, H, nKV, D, P, kind, apart, q_std=2.0, bar=False):
    """Groups of a few requests with a row each, one of many, and of chunks of rows."""
    if kind == "wide":
        widths, keys, own, added = [40], [500], np.arange(1, 41) * 5, 1
    elif kind == "chunks":
        widths, keys, own, added = [4, 2], [333, 90], [70, 40, 5, 33, 100, 65], [40, 13, 1, 0, 60, 30]
    else:
        widths, keys, own, added = [5, 3], [700, 40], [1, 2, 16, 33, 60, 300, 7, 64], 1
    c = shared_case(seed, dtype, H, nKV, D, P, widths, keys, own, added, q_std, apart)
    room = room_for_many(H, nKV, len(c[2])) if kind == "chunks" else 0
    got = attend(*c[:6], shared_names(kind, dtype, D, apart), room, kind == "chunks", groupStart=c[6], shared=c[7])
    q, row_start, lens, tables, k, v = c[:6]
    want = P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype), everything)
    check(got, want, D, q_std if bar else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("kind,apart", [("few", True), ("small", True), ("wide", True), ("chunks", True), ("few", False),
                                        ("small", False), ("chunks", False)])
@pytest.mark.parametrize("q_std", list(A.BARS))
def test_shared_accuracy(dtype, D, kind, apart, q_std):
    shared(D, dtype, 4, 2, D, 4 if kind == "small" else 16, kind, apart, q_std, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,nKV,D,P", [(6, 2, 24, 8), (9, 3, 72, 32), (10, 2, 80, 8), (12, 4, 104, 128), (20, 1, 120, 16), (33, 1, 40, 64),
                                       (70, 1, 32, 16)])
@pytest.mark.parametrize("apart", [True, False])
def test_chunks_behind_shared_keys(dtype, H, nKV, D, P, apart):
    shared(H + D, dtype, H, nKV, D, P, "chunks", apart)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,nKV,D", [(70, 1, 32), (140, 2, 16), (12, 1, 64), (100, 4, 72)])
def test_one_row_each_with_more_heads_than_a_block_has_columns(dtype, H, nKV, D):
    """Blocks of 64 columns for the shared keys, of 16 for the own ones."""
    shared(H, dtype, H, nKV, D, 16, "wide", True)


@pytest.mark.parametrize("dtype", TYPES)
def test_most_groups_by_the_kernel_of_many_columns(dtype):
    """The items' table of 4096 groups beside the stages."""
    rs = np.random.RandomState(4)
    n, H, D = 4096, 8, 8
    c = shared_case(3, dtype, H, 1, D, 8, np.ones(n, int), rs.randint(0, 20, n), rs.randint(1, 9, n), 1)
    got = attend(*c[:6], ["_shared_rows_%s_d64" % dtype, "_own_%s_d64_s" % dtype], 64 * n // H, groupStart=c[6], shared=c[7])
    q, row_start, lens, tables, k, v = c[:6]
    check(got, P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype), everything), D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("width,keys", [(2, 6000), (60, 900)])
def test_shared_keys_cut_before_chunks(dtype, D, width, keys):
    """Their partials are added by the kernel of many rows."""
    rs = np.random.RandomState(width)
    own = rs.randint(8, 60, width)
    c = shared_case(width, dtype, 4, 2, D, 16, [width], keys, own, np.minimum(own, rs.randint(1, 7, width)))
    q, row_start, lens, tables, k, v = c[:6]
    got = attend(*c[:6], shared_names("chunks", dtype, D, True), room_for_many(4, 2, width), groupStart=c[6], shared=c[7])
    check(got, P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype), everything), D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [40, 96, 128])
@pytest.mark.parametrize("junk", [np.nan, np.inf])
@pytest.mark.parametrize("apart", [True, False])
def test_chunks_and_what_is_not_finite(dtype, D, junk, apart):
    """Behind the requests' keys, and before the own ones in a copied page, nobody sees it; in
    an own key the request's later rows do, in a shared one all of the group."""
    H, nKV, P = 6, 2, 16
    c = shared_case(6, dtype, H, nKV, D, P, [3, 1], [37, 20], [30, 9, 40, 25], [5, 1, 20, 3], apart=apart)
    q, row_start, lens, tables, k, v, start, keys = c
    clean = [k.copy(), v.copy()]
    bad = {"f32": np.float32(junk), "f16": np.float16(junk),
           "bf16": np.uint16(np.float32(junk).view(np.uint32) >> 16 | (0x40 if np.isnan(junk) else 0))}[dtype]
    used = np.zeros((k.shape[0], P), bool)
    for b, n in enumerate(lens):
        t = np.arange(n)
        if b in (1, 2) and apart:  # (by themselves requests read their own copies)
            t = t[t >= 37]
        used[tables[b, t // P], t % P] = True
    for pool in (k, v):
        pool.transpose(0, 2, 1, 3)[~used] = bad
    names, room = shared_names("chunks", dtype, D, apart), room_for_many(H, nKV, 4)
    want = P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(clean[0], dtype), R.value(clean[1], dtype), everything)

    def run():
        return attend(*c[:6], names, room, groupStart=start, shared=keys)
    check(run(), want, D)
    t = lens[2] - 10
    at = tables[2, t // P], slice(None), t % P, 3
    keep = v[at].copy()
    v[at] = bad
    got, spoiled = run(), np.arange(row_start[3] - 10, row_start[3])
    assert not np.isfinite(got[spoiled][..., 3]).any()
    rest = np.delete(np.arange(len(q)), spoiled)
    check(got[rest], [x[rest] for x in want], D)
    v[at] = keep
    v[tables[0, 1], :, 5, 3] = bad
    got, n = run(), row_start[3]
    assert not np.isfinite(got[:n][..., 3]).any()
    check(got[n:], [x[n:] for x in want], D)
