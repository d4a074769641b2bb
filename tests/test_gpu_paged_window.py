"""Attention of rows that see a window of the last keys and the first ones, against 64 bits."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import pages_reference as P_
import paged_reference as R
from test_gpu_paged import attention_case, i32, last_error, placed, room_for_many, sync_error

pytestmark = pytest.mark.gpu


def visible(window, sinks):
    return lambda b, at, t: (t > at - window) | (t < sinks)


def drop(seed, tables, lens, added, P, window, sinks, n_pages):
    """Entries of pages that no row sees a key of: they may hold anything."""
    rs = np.random.RandomState(seed)
    out = tables.copy()
    for b, n in enumerate(lens):
        first = n - added[b]  # position of its first row
        for j in range(tables.shape[1]):
            if j * P >= n or (j * P >= sinks and (j + 1) * P - 1 <= first - window):
                out[b, j] = rs.choice([-1, n_pages, 2 ** 31 - 1, -2 ** 31, rs.randint(0, n_pages)])
    return out


def run(q, row_start, lens, tables, k, v, ragged, window, sinks, room=0, scale=0.0):
    rows, W = len(q), q.shape[1] * q.shape[2]
    room = max(room, rows)
    hq = np.full((room, W), np.nan, np.float32)
    hq[:rows] = q.reshape(rows, -1)
    out = R.upload(np.full((room, W), 5, np.float32))
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start) if ragged else None,
                     scale, out, window, sinks)
    device.sync()
    assert (out.data[rows:] == 5).all()
    return out.data[:rows]


def one(seed, dtype, H, nKV, D, P, lens, added, window, sinks, room=0, ragged=None):
    q, row_start, ln, tables, k, v = attention_case(seed, dtype, H, nKV, D, P, lens, added)
    tables = drop(seed, tables, ln, added, P, window, sinks, k.shape[0])
    ragged = any(a != 1 for a in added) or bool(room) if ragged is None else ragged
    got = run(q, row_start, ln, tables, k, v, ragged, window, sinks, room)
    want = P_.attention(q.astype(np.float64), row_start, ln, tables, R.value(k, dtype), R.value(v, dtype), visible(window, sinks))
    P_.check_attention(got, want, D)


TYPES = ["f32", "f16", "bf16"]
LENGTHS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 200, 257, 400, 513, 1000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (15, 0), (16, 16), (17, 3), (33, 33), (64, 64), (100, 4),
                                          (129, 70), (400, 1), (2000, 0), (1, 2000), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("P", [4, 16, 64])
def test_one_row_each(dtype, window, sinks, P):
    one(window % 89 + sinks % 83 + P, dtype, 4, 2, 32, P, LENGTHS, [1] * len(LENGTHS), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,nKV,D,P", [(1, 1, 8, 1), (9, 3, 64, 8), (10, 2, 80, 32), (12, 4, 96, 16), (20, 1, 128, 128), (33, 1, 40, 2)])
def test_heads_and_pages(dtype, H, nKV, D, P):
    one(H + D, dtype, H, nKV, D, P, [300, 41, 7, 150], [1] * 4, 50, 5)
    one(H + D, dtype, H, nKV, D, P, [300, 41, 7, 150], [3, 20, 7, 1], 50, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (16, 0), (40, 17), (64, 100), (90, 1), (333, 20), (5000, 4)])
@pytest.mark.parametrize("room", [0, room_for_many(6, 2, 5)])
@pytest.mark.parametrize("P", [8, 16, 128])
def test_ragged_rows(dtype, window, sinks, room, P):
    one(window + P, dtype, 6, 2, 24, P, [150, 30, 64, 400, 9], [150, 1, 20, 130, 0], window, sinks, room, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks,n", [(3000, 4, 9000), (5000, 700, 7000), (128, 2, 20000)])
def test_long_requests_are_cut(dtype, window, sinks, n):
    one(n, dtype, 8, 2, 64, 16, [n, n // 3], [1, 1], window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_chunk_of_a_long_prompt(dtype):
    """By the kernel of many rows, cut and joined."""
    one(3, dtype, 16, 2, 32, 32, [3000], [70], 1500, 40, room_for_many(16, 2, 1))
    one(4, dtype, 32, 2, 128, 16, [900, 500], [300, 20], 260, 4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [70, 300, 4096])
def test_many_requests(dtype, n):
    rs = np.random.RandomState(n)
    lens = rs.randint(0, 60 if n > 1000 else 300, n)
    one(n, dtype, 2, 1, 16, 8, lens, [1] * n, 21, 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_most_requests_with_many_columns(dtype):
    rs = np.random.RandomState(2)
    one(5, dtype, 8, 1, 8, 8, rs.randint(4, 40, 4096), [4] * 4096, 300, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ragged,room", [(False, 0), (True, 0), (True, room_for_many(6, 2, 4))])
@pytest.mark.parametrize("junk", [np.nan, np.inf, -np.inf])
def test_ignores_what_a_row_does_not_see(dtype, ragged, room, junk):
    """Keys between the sinks and the window, of dropped pages and behind a request
    hold what is not finite; so do keys that only some rows of a block see."""
    lens, added = [150, 40, 64, 300], ([2, 20, 64, 1] if ragged else [1] * 4)
    H, nKV, D, P, window, sinks = 6, 2, 72, 16, 23, 5
    q, row_start, ln, tables, k, v = attention_case(3, dtype, H, nKV, D, P, lens, added)
    clean = [k.copy(), v.copy()]
    bad = {"f32": np.float32(junk), "f16": np.float16(junk),
           "bf16": np.uint16(np.float32(junk).view(np.uint32) >> 16 | (0x40 if np.isnan(junk) else 0))}[dtype]
    used = np.zeros((k.shape[0], P), bool)
    for b, n in enumerate(lens):
        t = np.arange(n)
        t = t[(t > n - added[b] - window) | (t < sinks)]
        used[tables[b, t // P], t % P] = True
    for pool in (k, v):
        pool.transpose(0, 2, 1, 3)[~used] = bad
    spoiled = []
    if ragged:  # a key in the middle of the rows' windows: only those that see it
        for b, t in ((1, 30), (2, 20)):
            for pool in (k, v):
                pool[tables[b, t // P], :, t % P, 3] = bad
            first = ln[b] - added[b]
            spoiled += [row_start[b] + i for i in range(added[b]) if t <= first + i < t + window]
    got = run(q, row_start, ln, drop(3, tables, ln, added, P, window, sinks, k.shape[0]), k, v, ragged, window, sinks, room)
    got = got.reshape(q.shape)
    assert not np.isfinite(got[spoiled][..., 3]).any()
    want = P_.attention(q.astype(np.float64), row_start, ln, tables, R.value(clean[0], dtype), R.value(clean[1], dtype),
                        visible(window, sinks))
    rest = np.delete(np.arange(len(q)), spoiled)
    assert np.isfinite(got[rest]).all()
    P_.check_attention(got[rest], [x[rest] for x in want], D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 3)])
def test_a_window_of_everything_is_plain_attention(dtype, room):
    q, row_start, lens, tables, k, v = attention_case(8, dtype, 4, 2, 64, 16, [400, 33, 90], [50, 33, 1])
    W = [R.upload(x) for x in (k, v)]
    hq = np.zeros((max(room, len(q)), 256), np.float32)
    hq[:len(q)] = q.reshape(len(q), -1)
    args = (R.upload(hq), i32(lens), i32(tables), *W, i32(row_start))
    a, b = S.pagedAttention(*args), S.pagedAttention(*args, window=400)
    device.sync()
    x, y = a.data[:len(q)], b.data[:len(q)]
    assert np.linalg.norm(x - y) <= 2e-6 * np.linalg.norm(x)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_replayed_with_growing_requests(dtype):
    """A captured step: the lengths move, the windows with them."""
    ctx, H, nKV, D, P, window, sinks = device.ops_ctx(), 4, 2, 32, 16, 40, 3
    q, row_start, lens, tables, k, v = attention_case(9, dtype, H, nKV, D, P, [300, 200, 250], [1, 1, 1])
    ln, out = i32(lens), S.create([3, H * D])
    args = (R.upload(q.reshape(3, -1)), ln, i32(tables), R.upload(k), R.upload(v), None, 0.0, out, window, sinks)
    S.pagedAttention(*args)
    device.sync()
    device.check(device.lib.smith_graph_begin(ctx), "begin")
    S.pagedAttention(*args)
    g = device.lib.smith_graph_end(ctx)
    assert g, last_error()
    try:
        for now in ([10, 1, 250], [41, 200, 249], [300, 40, 0], [299, 17, 64]):
            ln.set_data(now)
            device.check(device.lib.smith_graph_launch(ctx, g))
            got = out.data
            want = P_.attention(q.astype(np.float64), row_start, now, tables, R.value(k, dtype), R.value(v, dtype),
                                visible(window, sinks))
            P_.check_attention(got, want, D)
            S.pagedAttention(*args[:7], None, 7, 1)  # eager, between
            device.sync()
    finally:
        device.lib.smith_graph_destroy(g)


@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 2)])
def test_a_page_outside_the_pool(room):
    q, row_start, lens, tables, k, v = attention_case(5, "f16", 4, 2, 32, 16, [140, 30], [1, 1])
    tables[0, 7] = -1  # in its window
    hq = np.zeros((max(room, 2), 128), np.float32)
    hq[:2] = q.reshape(2, -1)
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start), 0.0, None, 50, 2)
    assert "request 0: a page outside" in sync_error()
    device.sync()
    with pytest.raises(ValueError, match="a window of 0 keys and 3 sinks"):
        S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start), sinks=3)


def test_pages_beyond_32_bit_offsets():
    H, nKV, D, P = 8, 4, 64, 64
    n_pages = (5 << 30) // (nKV * P * D * 2)
    q, row_start, lens, tables, k, v = attention_case(17, "f16", H, nKV, D, P, [700, 130], [1, 70], spare=0)
    used = -(-lens // P)
    far = tables.copy()
    for b in range(2):
        tables[b, used[b]:] = 0
        far[b, :used[b]] = n_pages - 1 - tables[b, :used[b]]
    pools = [S.create([n_pages, nKV, P, D], "f16") for _ in range(2)]
    try:
        for t, host in zip(pools, (k, v)):
            for i in range(len(host)):
                device.upload(t.buffer + (n_pages - 1 - i) * host[i].nbytes, np.ascontiguousarray(host[i]))
        want = P_.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, "f16"), R.value(v, "f16"), visible(99, 9))
        for room in (len(q), room_for_many(H, nKV, 2)):
            hq = np.zeros((room, H * D), np.float32)
            hq[:len(q)] = q.reshape(len(q), -1)
            got = S.pagedAttention(R.upload(hq), i32(lens), i32(far), *pools, i32(row_start), window=99, sinks=9)
            device.sync()
            P_.check_attention(got.data[:len(q)], want, D)
    finally:
        for t in pools:
            t.release()


@pytest.mark.parametrize("over,message", [
    ({"kv": 3}, "unknown page type 3"), ({"window": 0}, "a window of 0 keys"), ({"H": 5}, "5 heads not a multiple of 2"),
    ({"D": 12}, "head_dim 12"), ({"max_pages": 0}, "block tables of 0"), ({"n_req": 4097, "max_rows": 4097}, "4097 requests"),
    ({"max_rows": 3}, "max_rows 3 for one row"), ({"ld_q": 63}, "row strides 63"), ({"k": None}, "page pools"),
    ({"lens": None}, "null buffer"), ({"out": 4096 + 256}, "out overlaps q"), ({"tables": 1 << 20}, "out overlaps an input"),
    ({"scale": float("nan")}, "scale nan")])
def test_refusals(over, message):
    a = dict(kv=1, q=4096, ld_q=64, max_rows=2, row_start=None, lens=4096, tables=4096, n_req=2, max_pages=4, window=9,
             sinks=0, H=4, nKV=2, D=16, scale=0.0, k=4096, v=4096, n_pages=8, P=16, out=1 << 20, ld_out=64)
    a.update(over)
    assert device.lib.smith_paged_attention_window(
        device.ops_ctx(), *placed(a, "q", "row_start", "lens", "tables", "k", "v", "out")) == -1
    assert "smith_paged_attention_window: " in last_error() and message in last_error()
