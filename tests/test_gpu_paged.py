"""The paged KV cache's operators against plain 64-bit forms: plan, append,
attention, and a run of them together."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import paged_reference as R

pytestmark = pytest.mark.gpu
# half a rounding step relative to the value
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def i32(a):
    return R.upload(np.asarray(a, np.int32))


def last_error():
    return device.lib.smith_last_error(device.ctx()).decode()


def sync_error():
    assert device.lib.smith_sync(device.ctx()) == -1
    return last_error()


# --------------------------------------------------------------------------
# plan
# --------------------------------------------------------------------------
def plan_inputs(seed, n, P, longest, most, spare_pages=3, spare_rows=0):
    rs = np.random.RandomState(seed)
    added = rs.randint(0, most + 1, n).astype(np.int32)
    cached = rs.randint(0, longest + 1, n).astype(np.int32)
    cached[rs.rand(n) < 0.3] //= P
    cached[rs.rand(n) < 0.3] *= 0
    old, new = -(-cached // P), -(-(cached + added) // P)
    max_pages = int(new.max()) + 2
    n_pages = int(new.sum()) + spare_pages
    order = rs.permutation(n_pages).astype(np.int32)
    tables = rs.randint(-5, 2 ** 30, (n, max_pages)).astype(np.int32)  # anything behind a request's pages
    at = 0
    for b in range(n):
        tables[b, :old[b]] = order[at:at + old[b]]
        at += old[b]
    free = order[at:]
    return cached, added, free, tables, n_pages, int(added.sum()) + spare_rows


def run_plan(cached, added, free, count, tables, n_pages, P, max_rows):
    t = i32(tables)
    plan = S.pagedPlan(i32(cached), i32(added), i32(free), i32([count]), t, n_pages, P, max_rows)
    return t, plan


@pytest.mark.parametrize("n,P,longest,most,spare_rows", [
    (1, 16, 0, 1, 0), (1, 16, 40, 0, 5), (1, 1, 7, 9, 0), (3, 2, 5, 4, 1), (24, 16, 300, 1, 8), (65, 32, 100, 70, 0),
    (255, 8, 50, 3, 255), (257, 64, 500, 20, 1), (700, 16, 90, 40, 0), (4096, 16, 33, 2, 300)])
def test_plan(n, P, longest, most, spare_rows):
    cached, added, free, tables, n_pages, max_rows = plan_inputs(n + P, n, P, longest, most, 3, spare_rows)
    want = R.plan(cached, added, free, len(free), tables, P, max_rows)
    got, plan = run_plan(cached, added, free, len(free), tables, n_pages, P, max(1, max_rows))
    device.sync()
    assert np.array_equal(got.data, want[0])
    assert np.array_equal(plan["rowStart"].data, want[1])
    assert np.array_equal(plan["lens"].data, want[2])
    assert np.array_equal(plan["slots"].data[:max_rows], want[3])
    assert np.array_equal(plan["positions"].data[:max_rows], want[4])
    assert plan["freeLeft"].data[0] == want[5]


def test_plan_takes_the_last_free_page():
    got, plan = run_plan(np.array([16], np.int32), np.array([17], np.int32), np.array([4, 1, 2], np.int32), 2,
                         np.array([[3, -1, -1]], np.int32), 5, 16, 17)
    device.sync()
    assert got.data.tolist() == [[3, 1, 4]] and plan["freeLeft"].data[0] == 0
    assert plan["slots"].data.tolist() == [1 * 16 + k for k in range(16)] + [4 * 16]


@pytest.mark.parametrize("what,message", [
    ("negative", "request 2: a length is negative"), ("long", "request 1: a length is negative or longer"),
    ("wraps", "request 0: a length is negative or longer"), ("rows", "more than max_rows = 9 rows"),
    ("pages", "more than the 1 free pages"), ("count", "free pages"), ("none", "more than the 0 free pages")])
def test_plan_that_does_not_fit_has_no_rows(what, message):
    cached = np.array([5, 16, 0, 31], np.int32)
    added = np.array([1, 3, 4, 2], np.int32)
    count, max_rows = 4, 10
    if what == "negative":
        added[2] = -4
    elif what == "long":
        added[1] = 49
    elif what == "wraps":
        cached[0] = added[0] = 2 ** 31 - 1
    elif what == "rows":
        max_rows = 9
    elif what == "pages":
        count = 1
    elif what == "count":
        count = 2 ** 31 - 1
    elif what == "none":
        count = 0
    tables = np.arange(16, dtype=np.int32).reshape(4, 4)
    got, plan = run_plan(cached, added, np.arange(20, 24), count, tables, 24, 16, max_rows)
    assert message in sync_error()
    device.sync()  # reported once
    assert np.array_equal(got.data, tables)
    assert not plan["rowStart"].data.any()
    assert (plan["slots"].data == -1).all() and (plan["positions"].data == -1).all()
    assert np.array_equal(plan["lens"].data, cached) and plan["freeLeft"].data[0] == count


@pytest.mark.parametrize("where", ["free", "table"])
@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1])
def test_plan_page_outside_the_pool(where, page):
    tables = np.array([[0, -1], [1, -1]], np.int32)
    free = np.array([4, 5], np.int32)
    if where == "free":
        free[0] = page  # request 1's new page
    else:
        tables[1, 0] = page
    _, plan = run_plan(np.array([16, 15], np.int32), np.array([1, 2], np.int32), free, 2, tables, 6, 16, 3)
    assert "request 1: a page outside the pool" in sync_error()
    want = [5 * 16, 31, -1] if where == "free" else [5 * 16, -1, 4 * 16]
    assert plan["slots"].data.tolist() == want


# --------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------
def rope_tables(n, seed):
    rs = np.random.RandomState(seed)
    a = rs.uniform(-3, 3, n)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def append_case(seed, dtype, H, nKV, D, rows, padding, P, rope, longest=50):
    rs = np.random.RandomState(seed)
    n_pages = -(-rows // P) + 3
    slots = rs.permutation(n_pages * P)[:rows].astype(np.int32)
    pos = rs.randint(0, longest, rows).astype(np.int32)
    pos[0] = longest - 1
    if padding:
        slots[rs.permutation(rows)[:padding]] = -1
    x = rs.standard_normal((rows, (H + 2 * nKV) * D)).astype(np.float32)
    half = {0: 0, 1: H * D // 2, 2: D // 2}[rope]
    cos, sin = rope_tables(longest * half, seed + 1)
    pools = [R.stored(rs.standard_normal((n_pages, nKV, P, D)), dtype) for _ in range(2)]
    return x, slots, pos, cos, sin, pools


def want_append(x, slots, pos, cos, sin, pools, dtype, H, nKV, D, P, rope):
    """(q, k pool, v pool) in f64 and the largest error of each element."""
    rows = len(x)
    q, k, v = x[:, :H * D], x[:, H * D:(H + nKV) * D], x[:, (H + nKV) * D:].astype(np.float64)
    if rope == 1:
        q, k = R.rotate(q, pos, cos, sin, H * D // 2), R.rotate(k, pos, cos, sin, nKV * D // 2)
    elif rope == 2:
        q, k = (R.rotate(y.reshape(rows, -1, D), pos, cos, sin, D // 2).reshape(rows, -1) for y in (q, k))
    # a product, a product and a sum in f32 (or fused: less): three half steps
    # of terms up to |x0| + |x1| <= 2 max|x|, |cos|, |sin| <= 1
    slack = 3 * HALF["f32"] * 2 * np.abs(x).max() if rope else 0.0
    out = []
    for y, pool, err in ((k, pools[0], slack), (v, pools[1], 0.0)):
        w = R.value(pool, dtype).copy()
        tol = np.zeros(w.shape)
        y = y.astype(np.float64).reshape(rows, nKV, D)
        for r, s in enumerate(slots):
            if s >= 0:
                w[s // P, :, s % P] = y[r]
                tol[s // P, :, s % P] = err + (HALF[dtype] * (np.abs(y[r]) + err) + 2.0 ** -25 if dtype != "f32" else 0.0)
        out.append((w, tol))
    return q.astype(np.float64), slack, out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rope", [0, 1, 2])
@pytest.mark.parametrize("H,nKV,D,rows,padding,P", [
    (4, 2, 16, 1, 0, 16), (4, 2, 16, 7, 3, 1), (9, 3, 64, 33, 0, 8), (8, 1, 128, 5, 5, 16), (10, 10, 40, 70, 11, 32),
    (32, 8, 128, 19, 2, 64), (1, 1, 8, 300, 0, 16)])
def test_append(dtype, rope, H, nKV, D, rows, padding, P):
    x, slots, pos, cos, sin, pools = append_case(rows + D, dtype, H, nKV, D, rows, padding, P, rope)
    kp, vp = (R.upload(p) for p in pools)
    q = S.pagedAppend(R.upload(x), i32(slots), i32(pos), H, kp, vp, rope, R.upload(cos) if rope else None,
                      R.upload(sin) if rope else None)
    device.sync()
    wq, slack, kv = want_append(x, slots, pos, cos, sin, pools, dtype, H, nKV, D, P, rope)
    there = slots >= 0
    assert np.all(np.abs(q.data[there] - wq[there]) <= slack)
    for t, (w, tol) in zip((kp, vp), kv):
        assert np.all(np.abs(R.value(t.data, dtype) - w) <= tol)


def raw_append(dtype, x_ptr, ld, rows, slots, pos, H, nKV, D, rope, cos, sin, n, kp, vp, n_pages, P, q_ptr, ld_q):
    return device.lib.smith_paged_append(device.ops_ctx(), S.paged.KV_TYPES[dtype], x_ptr, ld, rows, slots, pos, H, nKV,
                                         D, rope, cos, sin, n, kp, vp, n_pages, P, q_ptr, ld_q)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rope", [1, 2])
@pytest.mark.parametrize("shift,extra", [(0, 0), (0, 3), (1, 4), (3, 1)])
def test_append_strides_alignment_and_in_place(dtype, rope, shift, extra):
    """Rows `extra` floats further apart that start `shift` floats into their
    buffer, rotated in place; what lies between the rows stays."""
    H, nKV, D, rows, P = 6, 3, 24, 11, 4
    x, slots, pos, cos, sin, pools = append_case(shift + 5 * extra, dtype, H, nKV, D, rows, 2, P, rope)
    W = x.shape[1]
    ld = W + extra
    host = np.random.RandomState(3).standard_normal(shift + rows * ld).astype(np.float32)
    for r in range(rows):
        host[shift + r * ld:shift + r * ld + W] = x[r]
    buf, kp, vp = R.upload(host), R.upload(pools[0]), R.upload(pools[1])
    tc, ts, sl, po = R.upload(cos), R.upload(sin), i32(slots), i32(pos)
    at = buf.buffer + 4 * shift
    assert raw_append(dtype, at, ld, rows, sl.buffer, po.buffer, H, nKV, D, rope, tc.buffer, ts.buffer, cos.size,
                      kp.buffer, vp.buffer, pools[0].shape[0], P, at, ld) == 0, last_error()
    device.sync()
    wq, slack, kv = want_append(x, slots, pos, cos, sin, pools, dtype, H, nKV, D, P, rope)
    got = buf.data
    for r in range(rows):
        y = got[shift + r * ld:shift + (r + 1) * ld]
        if slots[r] >= 0:
            assert np.all(np.abs(y[:H * D] - wq[r]) <= slack)
            y[:H * D] = 0
            host[shift + r * ld:shift + r * ld + H * D] = 0
    assert np.array_equal(got, host)
    for t, (w, tol) in zip((kp, vp), kv):
        assert np.all(np.abs(R.value(t.data, dtype) - w) <= tol)


@pytest.mark.parametrize("dtype,x,want", [
    ("f16", [65519.0, 65520.0, -1e30, 2.0 ** -24, 2.0 ** -25, 1.0 + 2.0 ** -11, 1.0 + 3 * 2.0 ** -11, np.inf],
     [65504.0, np.inf, -np.inf, 2.0 ** -24, 0.0, 1.0, 1.0 + 2.0 ** -9, np.inf]),
    ("bf16", [3.38e38, 3.4e38, 1e-40, 2.0 ** -133, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, -np.inf, 0.0],
     [float((np.uint32(0x7F7E0000)).view(np.float32)), np.inf, None, 2.0 ** -133, 1.0, 1.0 + 2.0 ** -6, -np.inf, 0.0])])
def test_append_rounds_to_nearest_even(dtype, x, want):
    row = np.zeros((1, 24), np.float32)
    row[0, 16:] = x
    kp, vp = R.upload(R.stored(np.ones((1, 1, 2, 8)), dtype)), R.upload(R.stored(np.ones((1, 1, 2, 8)), dtype))
    S.pagedAppend(R.upload(row), i32([1]), i32([0]), 1, kp, vp)
    device.sync()
    got = R.value(vp.data, dtype)
    for g, w, v in zip(got[0, 0, 1], want, row[0, 16:]):
        assert g == (w if w is not None else R.value(R.to_bf16(np.array([v])), "bf16")[0])
    assert (got[0, 0, 0] == 1).all() and (R.value(kp.data, dtype)[0, 0, 0] == 1).all()


@pytest.mark.parametrize("bad,message", [
    ("slot", "row 2: its slot lies outside"), ("slot_low", "row 2: its slot lies outside"),
    ("position", "row 2: its position lies outside"), ("position_low", "row 2: its position lies outside")])
@pytest.mark.parametrize("rope", [1, 2])
def test_append_leaves_out_rows_that_do_not_fit(bad, message, rope):
    H, nKV, D, P, dtype = 4, 2, 16, 4, "f16"
    x, slots, pos, cos, sin, pools = append_case(9, dtype, H, nKV, D, 4, 0, P, rope)
    if bad.startswith("slot"):
        slots[2] = -2 if bad == "slot_low" else pools[0].shape[0] * P
    else:
        pos[2] = -1 if bad == "position_low" else 50
    kp, vp = R.upload(pools[0]), R.upload(pools[1])
    q = R.upload(np.full((4, H * D), 7, np.float32))
    tx, tc, ts, sl, po = R.upload(x), R.upload(cos), R.upload(sin), i32(slots), i32(pos)
    assert raw_append(dtype, tx.buffer, x.shape[1], 4, sl.buffer, po.buffer, H, nKV, D, rope, tc.buffer, ts.buffer,
                      cos.size, kp.buffer, vp.buffer, pools[0].shape[0], P, q.buffer, H * D) == 0
    assert message in sync_error()
    device.sync()
    slots[2], pos[2] = -1, 0
    wq, slack, kv = want_append(x, slots, pos, cos, sin, pools, dtype, H, nKV, D, P, rope)
    wq[2] = 7
    assert np.all(np.abs(q.data - wq) <= slack)
    for t, (w, tol) in zip((kp, vp), kv):
        assert np.all(np.abs(R.value(t.data, dtype) - w) <= tol)


def test_append_of_more_rows_than_a_grid_axis():
    """65600 rows take two launches; a slot outside the pool is reported by its row."""
    rs = np.random.RandomState(8)
    rows, P = 65600, 16
    x = rs.standard_normal((rows, 24)).astype(np.float32)
    slots = rs.permutation(rows).astype(np.int32)
    pools = [R.upload(np.zeros((rows // P, 1, P, 8), np.float16)) for _ in range(2)]
    tx, pos = R.upload(x), i32(np.zeros(rows))
    q = S.pagedAppend(tx, i32(slots), pos, 1, *pools)
    device.sync()
    assert np.array_equal(q.data, x[:, :8])
    for t, part in zip(pools, (x[:, 8:16], x[:, 16:])):
        assert np.array_equal(t.data.reshape(rows, 8)[slots], part.astype(np.float16))
    slots[65590] = rows
    S.pagedAppend(tx, i32(slots), pos, 1, *pools)
    assert "row 65590" in sync_error()


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------
def attention_case(seed, dtype, H, nKV, D, P, lens, added, q_std=2.0, spare=2):
    rs = np.random.RandomState(seed)
    lens, added = np.asarray(lens, np.int32), np.asarray(added, np.int32)
    pages = -(-lens // P)
    n_pages = max(1, int(pages.sum()) + spare)
    order = rs.permutation(n_pages).astype(np.int32)
    tables = rs.randint(-2 ** 31, 2 ** 31 - 1, (len(lens), int(pages.max()) + 1)).astype(np.int32)
    at = 0
    for b in range(len(lens)):
        tables[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
    k, v = (R.stored(rs.standard_normal((n_pages, nKV, P, D)), dtype) for _ in range(2))
    q = (rs.standard_normal((int(added.sum()), H, D)) * q_std).astype(np.float32)
    row_start = np.concatenate([[0], np.cumsum(added)]).astype(np.int32)
    return q, row_start, lens, tables, k, v


def check_attention(got, q, row_start, lens, tables, k, v, dtype, scale=None):
    """Each output against the 64-bit one.  A score is a sum of D products of q
    (kept to 2^-22 of its row's largest element) and k in f32: off by at most
    (D + 8) 2^-24 + 2^-21 of B = scale sum |q k|; its weight by twice that, and
    by 2^-21 for the exponential and the weight's own split; the sums over n keys by n half steps,
    each relative to sum p |v| / sum p."""
    want, mag, big = R.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype), scale)
    D = q.shape[2]
    rel = 2 * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) * big + 2.0 ** -20 + int(max(lens)) * 2.0 ** -23
    got = got.astype(np.float64).reshape(want.shape)
    off = np.abs(got - want)
    assert np.all(off <= mag * rel[..., None]), (off / (mag * rel[..., None] + 1e-300)).max()
    # roundings that are independent add up as their root: far below the bound of the sum
    norm = np.linalg.norm(want)
    if norm:
        assert np.linalg.norm(off) <= 1e-5 * norm, np.linalg.norm(off) / norm


def room_for_many(H, nKV, n_req):
    """max_rows with which the kernel of many rows answers: at least 8192 columns
    (row, head) and more than 24 of a KV head to a request."""
    return max(8192 // H, 24 * n_req * nKV // H) + 1


def run_attention(q, row_start, lens, tables, k, v, ragged, scale=0.0, room=0):
    """`room` rows in q and out, those behind the last sequence NaN in q; in out they stay."""
    rows, W = len(q), q.shape[1] * q.shape[2]
    room = max(room, rows)
    hq = np.full((room, W), np.nan, np.float32)
    hq[:rows] = q.reshape(rows, -1)
    out = R.upload(np.full((room, W), 5, np.float32))
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v),
                     i32(row_start) if ragged else None, scale, out)
    device.sync()
    assert (out.data[rows:] == 5).all()
    return out.data[:rows]


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 511, 513, 1000]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,nKV,D,P", [
    (4, 4, 64, 16), (16, 4, 64, 16), (32, 8, 128, 16), (8, 1, 128, 64), (9, 3, 64, 8), (10, 2, 80, 32), (12, 4, 96, 16),
    (3, 1, 8, 1), (2, 1, 16, 2), (40, 2, 40, 128), (17, 1, 120, 4), (6, 2, 88, 16), (4, 4, 80, 8), (7, 7, 72, 16)])
def test_attention_one_row_each(dtype, H, nKV, D, P):
    lens = LENGTHS if H * D < 2000 else LENGTHS[::3] + [129]
    case = attention_case(H + D + P, dtype, H, nKV, D, P, lens, [1] * len(lens))
    check_attention(run_attention(*case, ragged=False), *case, dtype)
    check_attention(run_attention(*case, ragged=True), *case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 17, 4097, 20011])
def test_attention_one_long_request(dtype, n):
    case = attention_case(n, dtype, 8, 2, 64, 32, [n], [1])
    check_attention(run_attention(*case, ragged=False), *case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,nKV,D,P,lens,added", [
    (4, 2, 64, 16, [1, 5, 40, 0, 70], [1, 5, 7, 0, 70]),          # prompts, a chunk, one that sits out
    (4, 1, 128, 8, [130, 65, 33], [67, 65, 1]),
    (8, 8, 64, 16, [100, 3], [100, 3]),                            # a head to a KV head
    (9, 3, 40, 4, [90, 17, 64], [50, 2, 64]),
    (32, 8, 128, 32, [75, 200], [33, 3]),
    (20, 1, 96, 16, [40, 41], [13, 41]),                           # more heads to a KV head than a tile has columns
    (2, 2, 8, 1, [30, 2, 9], [30, 1, 4]),
    (8, 1, 8, 16, [1500, 9], [1500, 2]),                           # more blocks than a wave has lanes
    (8, 2, 16, 32, [4000, 60, 700], [100, 60, 1]),                 # a chunk far behind its cache, cut, beside short ones
    (4, 4, 8, 16, [3000], [129]),
    (6, 2, 24, 16, [900, 900, 900], [900, 450, 31]),
    (4, 1, 128, 8, [300, 41], [250, 41]),                          # pages of half a wave's share of a stage
    (2, 2, 64, 8, [70, 200], [70, 111]),
    (4, 1, 32, 4, [130, 9], [130, 9]),
    (40, 1, 64, 16, [520, 7], [9, 7]),
    (4, 2, 80, 8, [90, 700, 5], [41, 30, 5]),
    (6, 2, 88, 16, [64, 1000], [64, 20]),
    (5, 5, 72, 32, [33, 65], [33, 1]),
    # more than 256 blocks, none cut: taken longest first
    (16, 16, 8, 16, [1000, 3, 90, 260, 0, 777, 128, 129], [1000, 3, 90, 260, 0, 777, 128, 129]),
    (16, 16, 8, 8, [900, 30, 600], [500, 30, 600]),
    (130, 1, 8, 16, [300, 40], [260, 40]),                         # several blocks to a row's heads
    (16, 4, 64, 64, [700], [9])])
def test_attention_ragged_rows(dtype, H, nKV, D, P, lens, added):
    case = attention_case(H + sum(lens), dtype, H, nKV, D, P, lens, added)
    check_attention(run_attention(*case, ragged=True), *case, dtype)
    check_attention(run_attention(*case, ragged=True, room=room_for_many(H, nKV, len(lens))), *case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_many_requests(dtype):
    rs = np.random.RandomState(4)
    lens = rs.randint(0, 60, 1100)
    added = np.minimum(rs.randint(0, 4, 1100), lens)
    case = attention_case(8, dtype, 4, 2, 16, 8, lens, added)
    check_attention(run_attention(*case, ragged=True), *case, dtype)
    check_attention(run_attention(*case, ragged=True, room=room_for_many(4, 2, 1100)), *case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_most_requests(dtype, D):
    """4096 requests, the most that are taken: the largest request table in LDS."""
    rs = np.random.RandomState(14)
    lens = rs.randint(0, 20, 4096)
    added = np.minimum(rs.randint(0, 3, 4096), lens)
    lens[4095], added[4095] = 700, 2
    case = attention_case(9, dtype, 2, 2, D, 16, lens, added)
    check_attention(run_attention(*case, ragged=True), *case, dtype)
    check_attention(run_attention(*case, ragged=True, room=room_for_many(2, 2, 4096)), *case, dtype)
    one = attention_case(10, dtype, 2, 2, D, 16, lens, [1] * 4096)
    check_attention(run_attention(*one, ragged=False), *one, dtype)


def replays(launch, out, case, dtype):
    """A captured call more than once, other work between: the same values each time."""
    ctx = device.ops_ctx()
    launch()
    device.sync()
    first = out.data.copy()
    device.check(device.lib.smith_graph_begin(ctx), "begin")
    launch()
    g = device.lib.smith_graph_end(ctx)
    assert g, last_error()
    try:
        for _ in range(4):
            out.set_data(np.full(first.shape, 5, np.float32))
            device.check(device.lib.smith_graph_launch(ctx, g))
            device.sync()
            assert np.array_equal(out.data, first)
            other = attention_case(3, dtype, 8, 2, 32, 16, [400, 30], [1, 20])
            check_attention(run_attention(*other, ragged=True), *other, dtype)
    finally:
        device.lib.smith_graph_destroy(g)
    check_attention(first[:len(case[0])], *case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ragged,lens,added", [
    (False, [900, 3, 40, 0, 2500] * 60, [1] * 300),        # 300 x 2 KV heads and more splits than workgroups
    (True, [700, 60, 1] * 50, [9, 60, 1] * 50),
    (True, [5000, 900, 33], [2000, 900, 33])])
def test_attention_more_items_than_workgroups_replayed(dtype, ragged, lens, added):
    """Workgroups that fetch further items off the queue, in a graph: what they
    count with is as it was when they end, and a joined sum has one order."""
    H, nKV = 8, 2
    case = q, row_start, lens, tables, k, v = attention_case(31, dtype, H, nKV, 16, 16, lens, added)
    rows = room_for_many(H, nKV, len(lens)) if ragged else len(q)
    hq = np.zeros((max(rows, len(q)), H * 16), np.float32)
    hq[:len(q)] = q.reshape(len(q), -1)
    tq, tl, tt, tk, tv, tr = R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(row_start)
    out = R.upload(np.full(hq.shape, 5, np.float32))
    replays(lambda: S.pagedAttention(tq, tl, tt, tk, tv, tr if ragged else None, 0.0, out), out, case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_request_without_keys_gives_zeros(dtype):
    case = attention_case(2, dtype, 4, 2, 32, 16, [0, 5, 0, 33, 0], [1] * 5)
    got = run_attention(*case, ragged=False)
    check_attention(got, *case, dtype)
    assert not got[[0, 2, 4]].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ragged,room", [(False, 0), (True, 0), (True, room_for_many(6, 2, 4))])
@pytest.mark.parametrize("junk", [np.nan, np.inf, -np.inf])
def test_attention_ignores_what_a_row_does_not_see(dtype, ragged, room, junk):
    """Slots behind a request's keys, pages of nobody and, for the rows before
    it, a later row's own key and value hold what is not finite."""
    lens, added = [5, 40, 64, 100], ([2, 20, 64, 1] if ragged else [1] * 4)
    H, nKV, D, P = 6, 2, 72, 16
    q, row_start, lens, tables, k, v = attention_case(3, dtype, H, nKV, D, P, lens, added)
    clean = R.stored(np.zeros(1), dtype)[0]
    bad = {"f32": np.float32(junk), "f16": np.float16(junk),
           "bf16": np.uint16(np.float32(junk).view(np.uint32) >> 16 | (0x40 if np.isnan(junk) else 0))}[dtype]
    used = np.zeros(k.shape[0] * P, bool)
    for b, n in enumerate(lens):
        used[(tables[b, np.arange(n) // P] * P + np.arange(n) % P)] = True
    hidden = ~used.reshape(k.shape[0], P)
    for pool in (k, v):
        pool.transpose(0, 2, 1, 3)[hidden] = bad
    if ragged:  # the last row of request 1 and 2 is not finite itself
        poisoned = []
        for b in (1, 2):
            t = lens[b] - 1
            for pool in (k, v):
                pool[tables[b, t // P], :, t % P, 3] = bad
            poisoned.append(row_start[b + 1] - 1)
        got = run_attention(q, row_start, lens, tables, k, v, True, room=room).reshape(q.shape)
        assert not np.isfinite(got[poisoned][..., 3]).any()
        for pool in (k, v):
            pool[~np.isfinite(R.value(pool, dtype))] = clean
        want, _, _ = R.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype))
        rest = np.delete(np.arange(len(q)), poisoned)
        assert np.linalg.norm(got[rest] - want[rest]) <= 1e-5 * np.linalg.norm(want[rest])
    else:
        got = run_attention(q, row_start, lens, tables, k, v, False)
        for pool in (k, v):
            pool.transpose(0, 2, 1, 3)[hidden] = clean
        check_attention(got, q, row_start, lens, tables, k, v, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e20])
@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 2)])
def test_attention_queries_of_any_size(dtype, size, room):
    """Queries far from 1 against a scale that brings the scores back."""
    q, row_start, lens, tables, k, v = attention_case(11, dtype, 4, 2, 64, 16, [300, 20], [3, 1])
    check_attention(run_attention(q * np.float32(size), row_start, lens, tables, k, v, True, 0.125 / size, room),
                    q * np.float32(size), row_start, lens, tables, k, v, dtype, 0.125 / size)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_far_scores(dtype, ragged):
    """One key far above the others, one far below, equal ones: weights of one, of
    nothing, and all alike."""
    q, row_start, lens, tables, k, v = attention_case(12, dtype, 2, 1, 16, 8, [100, 100, 64], [1, 1, 1])
    q[0] = 40.0
    q[2] = 0.0
    page = tables[0, 70 // 8]
    k[page, 0, 70 % 8] = R.stored(np.full(16, 3.0), dtype)
    got = run_attention(q, row_start, lens, tables, k, v, ragged, room=room_for_many(2, 1, 3) if ragged else 0)
    check_attention(got, q, row_start, lens, tables, k, v, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("spare", [9, room_for_many(6, 3, 3)])
def test_attention_strides_and_rows_behind_the_last(dtype, spare):
    """Row strides beyond the row, bases that are not 16-byte aligned, room for
    more rows than there are: everything else in out stays."""
    H, nKV, D, P = 6, 3, 56, 16
    q, row_start, lens, tables, k, v = attention_case(7, dtype, H, nKV, D, P, [20, 33, 50], [4, 1, 30])
    rows, W, room = len(q), H * D, len(q) + spare
    ld_q, ld_o = W + 3, W + 5
    hq = np.random.RandomState(1).standard_normal(1 + room * ld_q).astype(np.float32)
    ho = np.random.RandomState(2).standard_normal(3 + room * ld_o).astype(np.float32)
    for r in range(rows):
        hq[1 + r * ld_q:1 + r * ld_q + W] = q[r].ravel()
    tq, to, tk, tv = R.upload(hq), R.upload(ho), R.upload(k), R.upload(v)
    rs, ln, tb = i32(row_start), i32(lens), i32(tables)
    assert device.lib.smith_paged_attention(
        device.ops_ctx(), S.paged.KV_TYPES[dtype], tq.buffer + 4, ld_q, room, rs.buffer, ln.buffer, tb.buffer, 3,
        tables.shape[1], H, nKV, D, 0.0, tk.buffer, tv.buffer, k.shape[0], P, to.buffer + 12, ld_o) == 0, last_error()
    device.sync()
    got = to.data
    rows_at = [slice(3 + r * ld_o, 3 + r * ld_o + W) for r in range(rows)]
    check_attention(np.stack([got[s] for s in rows_at]), q, row_start, lens, tables, k, v, dtype)
    for s in rows_at:
        got[s] = ho[s]
    assert np.array_equal(got, ho)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad,message", [
    ("rows", "row_start ends at 3"), ("rows_low", "row_start ends at -1"), ("short", "request 1: its length"),
    ("long", "request 1: its length"), ("negative", "request 1: its length"), ("page", "request 1: a page outside"),
    ("page_low", "request 1: a page outside")])
@pytest.mark.parametrize("room", [2, room_for_many(4, 2, 2)])
def test_attention_leaves_out_what_does_not_fit(dtype, bad, message, room):
    q, row_start, lens, tables, k, v = attention_case(5, dtype, 4, 2, 32, 16, [40, 30], [1, 1])
    want, _, _ = R.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype))
    rs, ln, tb = row_start.copy(), lens.copy(), tables.copy()
    if bad == "rows":
        rs[2] = room + 1
        message = message.replace("3", str(room + 1))
    elif bad == "rows_low":
        rs[2] = -1
    elif bad == "short":
        ln[1] = 0
    elif bad == "long":
        ln[1] = tables.shape[1] * 16 + 1
    elif bad == "negative":
        ln[1] = -3
    else:
        tb[1, 1] = -1 if bad == "page_low" else k.shape[0]
    out = R.upload(np.full((room, 128), 5, np.float32))
    hq = np.zeros((room, 128), np.float32)
    hq[:2] = q.reshape(2, -1)
    S.pagedAttention(R.upload(hq), i32(ln), i32(tb), R.upload(k), R.upload(v), i32(rs), 0.0, out)
    assert message in sync_error()
    device.sync()
    got = out.data
    assert (got[2:] == 5).all()
    if bad.startswith("rows"):
        assert (got == 5).all()
    else:
        assert np.linalg.norm(got[0] - want[0].ravel()) <= 1e-5 * np.linalg.norm(want[0])
        if not bad.startswith("page"):
            assert (got[1] == 5).all()


@pytest.mark.parametrize("room", [4, room_for_many(4, 2, 3)])
def test_attention_row_start_out_of_order_stays_inside(room):
    """Starts that go back and forth between 0 and the total: no request has
    rows outside the buffers, and the calls after it are right."""
    case = attention_case(6, "f16", 4, 2, 32, 16, [40, 30, 20], [2, 1, 1])
    q, row_start, lens, tables, k, v = case
    run = (q, np.array([3, 1, 9, 4], np.int32), lens, tables, k, v)
    out, hq = R.upload(np.zeros((room, 128), np.float32)), np.zeros((room, 128), np.float32)
    hq[:4] = q.reshape(4, -1)
    S.pagedAttention(R.upload(hq), i32(lens), i32(tables), R.upload(k), R.upload(v), i32(run[1]), 0.0, out)
    assert "smith_paged_attention: request" in sync_error()
    check_attention(run_attention(*case, ragged=True, room=room), *case, "f16")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 2)])
@pytest.mark.parametrize("junk", [np.nan, np.inf])
def test_attention_of_a_query_that_is_not_finite(dtype, room, junk):
    """It spoils its own row's head and nothing else."""
    case = q, row_start, lens, tables, k, v = attention_case(19, dtype, 4, 2, 64, 16, [150, 40], [37, 3])
    clean = run_attention(*case, ragged=True, room=room).reshape(q.shape)
    q[5, 1, 7] = junk
    got = run_attention(*case, ragged=True, room=room).reshape(q.shape)
    assert not np.isfinite(got[5, 1]).any()
    got[5, 1] = clean[5, 1]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_graphs_on_one_scratch(dtype):
    """A captured step of prompts and one of single rows, replayed in turn."""
    ctx, H, nKV, D = device.ops_ctx(), 8, 2, 32
    steps = []
    for lens, added, ragged in (([900, 300, 80], [900, 300, 80], True), ([3000, 700, 41], [1, 1, 1], False)):
        case = q, row_start, ln, tables, k, v = attention_case(23, dtype, H, nKV, D, 16, lens, added)
        rows = max(len(q), room_for_many(H, nKV, 3)) if ragged else len(q)
        hq = np.zeros((rows, H * D), np.float32)
        hq[:len(q)] = q.reshape(len(q), -1)
        args = [R.upload(hq), i32(ln), i32(tables), R.upload(k), R.upload(v), i32(row_start) if ragged else None, 0.0,
                S.create([rows, H * D])]
        S.pagedAttention(*args)
        device.sync()
        steps.append([case, args, args[-1].data.copy(), None])
        check_attention(steps[-1][2][:len(q)], *case, dtype)
    try:
        for st in steps:
            device.check(device.lib.smith_graph_begin(ctx), "begin")
            S.pagedAttention(*st[1])
            st[3] = device.lib.smith_graph_end(ctx)
            assert st[3], last_error()
        for _ in range(4):
            for case, args, want, g in steps:
                args[-1].set_data(np.zeros(want.shape, np.float32))
            for case, args, want, g in steps:
                device.check(device.lib.smith_graph_launch(ctx, g))
            for case, args, want, g in steps:
                assert np.array_equal(args[-1].data[:len(case[0])], want[:len(case[0])])
    finally:
        for st in steps:
            if st[3]:
                device.lib.smith_graph_destroy(st[3])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_pages_beyond_32_bit_offsets(dtype):
    """Pools of 5 GiB: rows appended into their last pages, and attention over
    them by both kernels.  Only the pages of the requests are ever written."""
    H, nKV, D, P = 8, 4, 64, 64
    page = nKV * P * D
    n_pages = (5 << 30) // (page * (4 if dtype == "f32" else 2))
    lens, added = np.array([200, 65, 130], np.int32), np.array([200, 1, 70], np.int32)
    case = attention_case(17, dtype, H, nKV, D, P, lens, added, spare=0)
    q, row_start, _, tables, k, v = case
    used = -(-lens // P)
    for b in range(3):
        tables[b, used[b]:] = -1
    far = np.where(tables >= 0, n_pages - 1 - tables, tables)
    pools = [S.create([n_pages, nKV, P, D], dtype) for _ in range(2)]
    try:
        size = page * k.itemsize
        for t, host in zip(pools, (k, v)):
            for i in range(len(host)):
                device.upload(t.buffer + (n_pages - 1 - i) * size, np.ascontiguousarray(host[i]))
        rs = np.random.RandomState(3)
        # request 2's last row anew, through append
        x = rs.standard_normal((1, (H + 2 * nKV) * D)).astype(np.float32)
        slot = far[2, 129 // P].astype(np.int64) * P + 129 % P
        assert slot * nKV * D * k.itemsize > 1 << 32
        S.pagedAppend(R.upload(x), i32([slot]), i32([129]), H, *pools)
        for host, part in ((k, x[0, H * D:(H + nKV) * D]), (v, x[0, (H + nKV) * D:])):
            host[tables[2, 129 // P], :, 129 % P] = R.stored(part, dtype).reshape(nKV, D)
        for room in (len(q), room_for_many(H, nKV, 3)):
            hq = np.zeros((room, H * D), np.float32)
            hq[:len(q)] = q.reshape(len(q), -1)
            got = S.pagedAttention(R.upload(hq), i32(lens), i32(far), *pools, i32(row_start))
            device.sync()
            check_attention(got.data[:len(q)], q, row_start, lens, tables, k, v, dtype)
    finally:
        for t in pools:
            t.release()


# --------------------------------------------------------------------------
# refusals (nothing is launched); addresses are places in one buffer of zeros
# --------------------------------------------------------------------------
_arena = []


def placed(args, *pointers):
    if not _arena:
        _arena.append(S.zeros([1 << 20], "i32"))
    return [_arena[0].buffer + v if k in pointers and v is not None else v for k, v in args.items()]


def base_attention(**over):
    # pools of 8 pages x 2 heads x 16 keys x 16 dims of 2 bytes: 8192 bytes
    a = dict(kv=1, q=4096, ld_q=64, max_rows=2, row_start=None, lens=4096, tables=4096, n_req=2, max_pages=4, H=4, nKV=2,
             D=16, scale=0.0, k=4096, v=4096, n_pages=8, P=16, out=1 << 20, ld_out=64)
    a.update(over)
    return device.lib.smith_paged_attention(device.ops_ctx(), *placed(a, "q", "row_start", "lens", "tables", "k", "v", "out"))


@pytest.mark.parametrize("over,message", [
    ({"kv": 3}, "unknown page type 3"), ({"H": 5}, "5 heads not a multiple of 2"), ({"H": 0}, "0 heads"),
    ({"nKV": 0}, "of 0 kv heads"), ({"D": 0}, "head_dim 0"), ({"D": 12}, "head_dim 12"), ({"D": 136}, "head_dim 136"),
    ({"P": 0}, "page size 0"), ({"P": 24}, "page size 24"), ({"n_pages": 0}, "pool of 0 pages"),
    ({"n_pages": 1 << 27}, "pool of"), ({"max_pages": 0}, "block tables of 0"), ({"max_pages": 1 << 27}, "block tables of"),
    ({"n_req": 0, "max_rows": 0}, "0 requests"), ({"n_req": 4097, "max_rows": 4097}, "4097 requests"),
    ({"max_rows": 3}, "max_rows 3 for one row"), ({"ld_q": 63}, "row strides 63"), ({"ld_out": 60}, "and 60"),
    ({"k": None}, "page pools"), ({"v": 4104}, "16-byte aligned"), ({"q": None}, "null buffer"), ({"lens": None}, "null buffer"),
    ({"tables": None}, "null buffer"), ({"out": None}, "null buffer"), ({"out": 4096 + 256}, "out overlaps q"),
    ({"lens": (1 << 20) + 8}, "out overlaps an input"), ({"tables": 1 << 20}, "out overlaps an input"),
    ({"k": (1 << 20) - 8176}, "out overlaps an input"), ({"v": (1 << 20) + 256}, "out overlaps an input"),
    ({"row_start": 1 << 20}, "out overlaps an input"),
    ({"scale": float("nan")}, "scale nan"), ({"scale": float("inf")}, "scale inf"),
    ({"row_start": 4096, "max_rows": 1 << 31}, "max_rows 2147483648")])
def test_attention_refusals(over, message):
    assert base_attention(**over) == -1
    assert "smith_paged_attention: " in last_error() and message in last_error()


def base_append(**over):
    a = dict(kv=1, x=4096, ld=128, rows=2, slots=4096, pos=4096, H=4, nKV=2, D=16, rope=2, cos=4096, sin=4096, n=80,
             k=4096, v=4096, n_pages=8, P=16, q=1 << 20, ld_q=64)
    a.update(over)
    return device.lib.smith_paged_append(device.ops_ctx(), *placed(a, "x", "slots", "pos", "cos", "sin", "k", "v", "q"))


@pytest.mark.parametrize("over,message", [
    ({"kv": 9}, "unknown page type 9"), ({"H": 3}, "3 heads"), ({"D": 20}, "head_dim 20"), ({"P": 3}, "page size 3"),
    ({"rope": 3}, "unknown rotary indexing 3"), ({"cos": None}, "need both tables"), ({"q": None}, "need both tables and q_out"),
    ({"ld": 127}, "row strides 127"), ({"ld_q": 63}, "and 63"), ({"x": None}, "null buffer"), ({"slots": None}, "null buffer"),
    ({"pos": None}, "null buffer"), ({"rows": 1 << 31}, "rows"), ({"q": 4096 + 64}, "overlaps qkv"),
    ({"q": 4096, "ld_q": 64}, "overlaps qkv"), ({"k": 4100}, "16-byte aligned"), ({"v": None}, "page pools"),
    ({"k": 1 << 17, "v": (1 << 17) + 8176}, "two outputs overlap"), ({"v": 1 << 17}, "overlaps an input"),
    ({"k": 1 << 17, "v": 1 << 18, "q": 1 << 18}, "two outputs overlap"),
    ({"k": 1 << 17, "v": 1 << 18, "slots": 1 << 17}, "overlaps an input"),
    ({"k": 1 << 17, "v": 1 << 18, "sin": (1 << 20) + 4}, "overlaps an input")])
def test_append_refusals(over, message):
    assert base_append(**over) == -1
    assert "smith_paged_append: " in last_error() and message in last_error()


def base_plan(**over):
    a = dict(cached=0x1000, added=0x2000, n=4, free=0x3000, count=0x4000, n_pages=8, P=16, max_pages=4, max_rows=8,
             tables=0x5000, row_start=0x6000, lens=0x7000, slots=0x8000, positions=0x9000, left=0xA000)
    a.update(over)
    return device.lib.smith_paged_plan(device.ops_ctx(), *placed(a, "cached", "added", "free", "count", "tables", "row_start",
                                                                 "lens", "slots", "positions", "left"))


@pytest.mark.parametrize("over,message", [
    ({"n": 0}, "0 requests"), ({"n": 4097}, "4097 requests"), ({"P": 0}, "page size 0"), ({"P": 12}, "page size 12"),
    ({"n_pages": 0}, "pool of 0"), ({"max_pages": 0}, "max_pages 0"), ({"max_pages": 1 << 28}, "block tables"),
    ({"max_rows": 1 << 31}, "max_rows"), ({"lens": 0x1000}, "overlaps an input"), ({"left": 0x4000}, "overlaps an input"),
    ({"row_start": 0x200C}, "overlaps an input"), ({"slots": 0x9010}, "two outputs overlap"), ({"lens": 0x5030}, "two outputs"),
    ({"cached": None}, "null buffer"), ({"slots": None}, "null buffer"), ({"left": None}, "null buffer")])
def test_plan_refusals(over, message):
    assert base_plan(**over) == -1
    assert "smith_paged_plan: " in last_error() and message in last_error()


def test_calls_of_no_rows():
    assert base_append(rows=0, x=None, slots=None, pos=None) == 0
    assert base_attention(row_start=4096, max_rows=0, q=None, out=None) == 0
    device.sync()


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------
class Server:
    """A few requests on one layer, step by step, and their keys in f64."""

    def __init__(self, seed, n, dtype, H=8, nKV=2, D=32, P=16, max_pages=8, max_rows=96):
        self.rs, self.n, self.dtype, self.H, self.nKV, self.D, self.P, self.max_rows = (
            np.random.RandomState(seed), n, dtype, H, nKV, D, P, max_rows)
        n_pages = n * max_pages
        self.n_pages = n_pages
        self.pools = [R.upload(R.stored(np.full((n_pages, nKV, P, D), np.nan), dtype) if dtype != "bf16" else
                               np.full((n_pages, nKV, P, D), 0x7FC0, np.uint16)) for _ in range(2)]
        self.tables = i32(np.full((n, max_pages), -1))
        self.free = i32(self.rs.permutation(n_pages))
        self.cached, self.count = i32(np.zeros(n)), i32([n_pages])
        self.cos, self.sin = rope_tables(max_pages * P * D // 2, seed)
        self.tc, self.ts = R.upload(self.cos), R.upload(self.sin)
        self.keys = [[np.zeros((nKV, 0, D)), np.zeros((nKV, 0, D))] for _ in range(n)]

    def rows(self, added):
        return self.rs.standard_normal((self.max_rows, (self.H + 2 * self.nKV) * self.D)).astype(np.float32)

    def launch(self, x, added):
        plan = S.pagedPlan(self.cached, added, self.free, self.count, self.tables, self.n_pages, self.P, self.max_rows)
        q = S.pagedAppend(x, plan["slots"], plan["positions"], self.H, *self.pools, S.ROPE_HEAD, self.tc, self.ts)
        out = S.pagedAttention(q, plan["lens"], self.tables, *self.pools, plan["rowStart"])
        return plan, q, out

    def want(self, x, added):
        """The rows' outputs from the dense keys; takes the new ones in."""
        H, nKV, D, out, r = self.H, self.nKV, self.D, [], 0
        for b, n in enumerate(added):
            if not n:
                continue
            y = x[r:r + n]
            pos = self.keys[b][0].shape[1] + np.arange(n)
            q = R.rotate(y[:, :H * D].reshape(n, H, D), pos, self.cos, self.sin, D // 2)
            k = R.rotate(y[:, H * D:(H + nKV) * D].reshape(n, nKV, D), pos, self.cos, self.sin, D // 2)
            v = y[:, (H + nKV) * D:].reshape(n, nKV, D)
            for s, new in enumerate((k, v)):
                kept = R.value(R.stored(new, self.dtype), self.dtype)
                self.keys[b][s] = np.concatenate([self.keys[b][s], kept.transpose(1, 0, 2)], 1)
            kk, vv = (a[:, None] for a in self.keys[b])  # pages of one request's whole length
            o, _, _ = R.attention(q, [0, n], [kk.shape[2]], np.zeros((1, 1), int), kk.transpose(1, 0, 2, 3),
                                  vv.transpose(1, 0, 2, 3))
            out.append(o)
            r += n
        return np.concatenate(out).reshape(r, -1), r


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("max_rows", [96, room_for_many(8, 2, 6)])
def test_steps_of_several_requests(dtype, max_rows):
    """Prompts, then chunks and single rows, one request sitting out now and
    then; nothing waits between a step's three calls.  A key that rounds the
    other way in 64 bits is off by a step of its type (f16 2^-10) in one of
    32 dims of one key: 2e-3 of the norm holds many of them, not a wrong key."""
    sv = Server(5, 6, dtype, max_rows=max_rows)
    for step, added in enumerate(([20, 1, 33, 0, 17, 5], [1, 1, 1, 40, 0, 1], [1, 50, 1, 1, 16, 0], [1] * 6, [0, 0, 1, 1, 1, 1])):
        x = sv.rows(added)
        plan, _, out = sv.launch(R.upload(x), i32(added))
        device.sync()
        want, n = sv.want(x, added)
        err = np.linalg.norm(out.data[:n] - want) / np.linalg.norm(want)
        assert err <= {"f32": 1e-5, "f16": 2e-3, "bf16": 2e-3}[dtype], (step, err)
        sv.cached, sv.count = plan["lens"], plan["freeLeft"]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("max_rows", [96, room_for_many(8, 2, 5)])
def test_captured_decode_steps(dtype, max_rows):
    """A captured step of one row each, fed by its own lengths, replayed with
    other work between the replays: each replay equals the eager step."""
    a, b = Server(7, 5, dtype, max_rows=max_rows), Server(7, 5, dtype, max_rows=max_rows)
    ctx = device.ops_ctx()
    first = [30, 3, 16, 1, 40]
    x = a.rows(first)
    for s in (a, b):
        plan, _, _ = s.launch(R.upload(x), i32(first))
        s.cached, s.count = plan["lens"], plan["freeLeft"]
    ones, xin = i32([1] * 5), R.upload(np.zeros_like(x))
    q, out = S.create([a.max_rows, a.H * a.D]), S.create([a.max_rows, a.H * a.D])
    plan = {n: S.create([m], "i32") for n, m in (("rowStart", 6), ("lens", 5), ("slots", a.max_rows),
                                                 ("positions", a.max_rows), ("freeLeft", 1))}
    kv = S.paged.KV_TYPES[dtype]

    def step(s):
        L = device.lib
        device.check(L.smith_paged_plan(ctx, s.cached.buffer, ones.buffer, 5, s.free.buffer, s.count.buffer, s.n_pages, s.P,
                                        8, s.max_rows, s.tables.buffer, *(plan[n].buffer for n in
                                        ("rowStart", "lens", "slots", "positions", "freeLeft"))))
        device.check(L.smith_paged_append(ctx, kv, xin.buffer, x.shape[1], s.max_rows, plan["slots"].buffer,
                                          plan["positions"].buffer, s.H, s.nKV, s.D, 2, s.tc.buffer, s.ts.buffer, s.tc.size,
                                          s.pools[0].buffer, s.pools[1].buffer, s.n_pages, s.P, q.buffer, s.H * s.D))
        device.check(L.smith_paged_attention(ctx, kv, q.buffer, s.H * s.D, s.max_rows, plan["rowStart"].buffer,
                                             plan["lens"].buffer, s.tables.buffer, 5, 8, s.H, s.nKV, s.D, 0.0,
                                             s.pools[0].buffer, s.pools[1].buffer, s.n_pages, s.P, out.buffer, s.H * s.D))
        device.check(L.smith_copy_d2d(ctx, s.cached.buffer, 0, plan["lens"].buffer, 0, 20))
        device.check(L.smith_copy_d2d(ctx, s.count.buffer, 0, plan["freeLeft"].buffer, 0, 4))

    xs = [a.rows([1] * 5) for _ in range(6)]
    eager = []
    for y in xs:
        xin.set_data(y)
        step(a)
        eager.append(out.data[:5].copy())
    xin.set_data(xs[0])
    step(b)
    assert np.array_equal(out.data[:5], eager[0])
    device.check(device.lib.smith_graph_begin(ctx), "begin")
    step(b)
    g = device.lib.smith_graph_end(ctx)
    assert g, last_error()
    try:
        for y, want in zip(xs[1:], eager[1:]):
            xin.set_data(y)
            device.check(device.lib.smith_graph_launch(ctx, g))
            got = out.data[:5].copy()
            assert np.array_equal(got, want)
            # eager work of another size between the replays, on the same scratch
            case = attention_case(3, dtype, 8, 2, 32, 16, [400, 30], [1, 20])
            check_attention(run_attention(*case, ragged=True), *case, dtype)
    finally:
        device.lib.smith_graph_destroy(g)


def test_two_contexts():
    """The same call on two contexts' streams at once."""
    other = device.lib.smith_init()
    try:
        for path in (device.CODE_OBJECT_PATH, device.LLAMA_CODE_OBJECT_PATH, device.GEMM_CODE_OBJECT_PATH,
                     device.PAGED_CODE_OBJECT_PATH):
            assert device.lib.smith_load_library(other, path.encode())
        q, row_start, lens, tables, k, v = attention_case(21, "f16", 8, 2, 64, 16, [3000, 800, 5], [1, 1, 1])
        tq, tk, tv, tl, tt = R.upload(q.reshape(3, -1)), R.upload(k), R.upload(v), i32(lens), i32(tables)
        outs = [[S.create([3, 512]) for _ in range(4)] for _ in range(2)]
        device.sync()
        for i in range(4):
            for c, o in ((device.ops_ctx(), outs[0][i]), (other, outs[1][i])):
                assert device.lib.smith_paged_attention(c, 1, tq.buffer, 512, 3, None, tl.buffer, tt.buffer, 3, tables.shape[1],
                                                        8, 2, 64, 0.0, tk.buffer, tv.buffer, k.shape[0], 16, o.buffer, 512) == 0
        device.sync()
        assert device.lib.smith_sync(other) == 0
        for o in outs[0] + outs[1]:
            check_attention(o.data, q, row_start, lens, tables, k, v, "f16")
    finally:
        device.lib.smith_destroy(other)
