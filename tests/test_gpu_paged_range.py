"""Paged attention where weights, keys or values span far: what f32 arithmetic
holds of them is held, and what f16 pages lose is no more than is stated."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import attention_case, check_attention, room_for_many, run_attention

pytestmark = pytest.mark.gpu


def weights(q, row_start, lens, tables, k, v, dtype, scale=None):
    """(sum of the weights relative to the largest, sum of |v| of the keys that are
    seen, sum of weight times |v|), [rows, heads(, dim)] in f64."""
    H, D = q.shape[1:]
    G = H // k.shape[1]
    scale = D ** -0.5 if not scale else scale
    kf, vf = R.value(k, dtype), R.value(v, dtype)
    sw, sv, swv = np.zeros(q.shape[:2]), np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(lens):
        r0, r1 = row_start[b], row_start[b + 1]
        kk, vv = R.gathered(kf, tables[b], n), np.abs(R.gathered(vf, tables[b], n))
        for r in range(r0, r1):
            t = n - (r1 - r0) + (r - r0) + 1
            for h in range(H):
                s = scale * (kk[h // G, :t] @ q[r, h].astype(np.float64))
                w = np.exp(s - s.max())
                sw[r, h], sv[r, h], swv[r, h] = w.sum(), vv[h // G, :t].sum(0), w @ vv[h // G, :t]
    return sw, sv, swv


# (columns of one kernel or of the other, rows of a request or one, pages of less than 16 keys)
FORMS = [(False, 0, 16), (True, 0, 16), (True, room_for_many(4, 2, 3), 16), (False, 0, 4), (True, room_for_many(4, 2, 3), 8)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ragged,room,P", FORMS)
@pytest.mark.parametrize("size", [1e-35, 1e-20, 1e30])
def test_queries_far_from_one(dtype, ragged, room, P, size):
    H, nKV, D = 4, 2, 64
    q, row_start, lens, tables, k, v = attention_case(44, dtype, H, nKV, D, P, [300, 64, 41], [3, 1, 2] if ragged else [1, 1, 1])
    q = (np.copysign(1 + np.abs(q), q) * size).astype(np.float32)
    scale = float(np.float32(0.125 / size))
    case = q, row_start, lens, tables, k, v
    check_attention(run_attention(*case, ragged=ragged, scale=scale, room=room), *case, dtype, scale)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ragged,room,P", FORMS)
@pytest.mark.parametrize("size", [1e4, 1e6, 1e7, 1e8, 1e9, 1e12])
def test_scores_of_any_size(dtype, ragged, room, P, size):
    """Scores so far up that f32's next number is another weight: the best key is
    all there is, keys alike weigh alike, and nothing overflows on the way."""
    H, nKV, D = 4, 2, 64
    q, row_start, lens, tables, k, v = attention_case(45, dtype, H, nKV, D, P, [300, 64, 41], [3, 1, 2] if ragged else [1, 1, 1])
    for sign in (1.0, -1.0):
        if sign < 0:  # the scores of a row below zero, all but one dim of its keys 0
            q[..., 0] = np.abs(q[..., 0]) + 1
            flat = R.value(k, dtype)
            flat[..., 1:] = 0
            flat[..., 0] = -1 - np.abs(flat[..., 0])
            k = R.stored(flat, dtype)
        far = (q * size).astype(np.float32)
        case = far, row_start, lens, tables, k, v
        got = run_attention(*case, ragged=ragged, room=room)
        assert np.isfinite(got).all()
        got = got.astype(np.float64).reshape(q.shape)
        # whatever the scores' roundings choose among the best keys: a mean of their values
        kf, vf = R.value(k, dtype), R.value(v, dtype)
        for b, n in enumerate(lens):
            kk, vv = R.gathered(kf, tables[b], n), R.gathered(vf, tables[b], n)
            for r in range(row_start[b], row_start[b + 1]):
                t = n - (row_start[b + 1] - row_start[b]) + (r - row_start[b]) + 1
                for h in range(H):
                    s = D ** -0.5 * (kk[h // 2, :t] @ far[r, h].astype(np.float64))
                    # a score is off by (D + 10) half steps of its terms' size at most, twice that between two;
                    # 40 further down a weight is less than 2^-57
                    reach = 2 * (D + 10) * 2.0 ** -24 * D ** -0.5 * (np.abs(kk[h // 2, :t]) @ np.abs(far[r, h].astype(np.float64))).max() + 40
                    best = vv[h // 2, :t][s >= s.max() - reach]
                    slack = 1e-5 * np.abs(best).max(0)
                    assert (got[r, h] >= best.min(0) - slack).all() and (got[r, h] <= best.max(0) + slack).all(), (b, r, h)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("above", [12.0, 24.4, 30.4, 36.0])
@pytest.mark.parametrize("at", [0, 70])
@pytest.mark.parametrize("ragged,room,P", FORMS)
def test_small_weights_beside_a_dominating_key(dtype, above, at, ragged, room, P):
    """A key `above` powers of two over the others whose value is 0: the output is
    made of the small weights alone.  f32 and bf16 pages hold each to f32's
    accuracy.  f16 pages hold a weight to 2^-22 of itself and 2^-38 of the
    largest: P is 2^13 or more there, in two f16 parts whose second rounds at
    2^-25, half of f16's least step."""
    H, nKV, D = 4, 2, 64
    added = [3, 1, 20] if ragged else [1, 1, 1]
    q, row_start, lens, tables, k, v = attention_case(41, dtype, H, nKV, D, P, [150, 90, 300], added, q_std=0.1)
    rs = np.random.RandomState(5)
    u = np.where(rs.rand(D) < 0.5, -1.0, 1.0)
    q += u.astype(np.float32)  # all queries point along u, more or less
    far = above * np.log(2.0) / D ** 0.5 * u  # scale q.k is about above * ln 2
    for b in range(3):
        page = tables[b, at // P]
        k[page, :, at % P] = R.stored(np.broadcast_to(far, (nKV, D)), dtype)
        v[page, :, at % P] = R.stored(np.zeros((nKV, D)), dtype)
    got = run_attention(q, row_start, lens, tables, k, v, ragged, room=room).reshape(q.shape).astype(np.float64)
    want, mag, big = R.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype))
    # the bound of check_attention, and the floor of f16's weights
    rel = 2 * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) * big + 2.0 ** -20 + int(max(lens)) * 2.0 ** -23
    bound = mag * rel[..., None]
    if dtype == "f16":
        sw, sv, _ = weights(q, row_start, lens, tables, k, v, dtype)
        bound += 2.0 ** -38 * sv / sw[..., None]
    off = np.abs(got - want)
    assert np.all(off <= bound), (off / bound).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ragged,room,P", FORMS)
@pytest.mark.parametrize("split", [False, True])
def test_values_up_to_the_end_of_f32(dtype, ragged, room, P, split):
    """Values whose weighted sum, of weights up to 1, is just inside f32."""
    H, nKV, D = 4, 2, 64
    lens = [3000, 700, 41] if split else [100, 64, 41]
    case = attention_case(42, dtype, H, nKV, D, P, lens, [3, 1, 2] if ragged else [1, 1, 1])
    q, row_start, lens, tables, k, v = case
    _, _, swv = weights(*case, dtype)
    v = R.stored(R.value(v, dtype) * (2.0 ** 127 / swv.max()), dtype)
    case = q, row_start, lens, tables, k, v
    check_attention(run_attention(*case, ragged=ragged, room=room), *case, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ragged,room,P", FORMS)
def test_values_near_the_least_of_f32(dtype, ragged, room, P):
    """Values of 1e-36, which weights of 2^-8 and less make subnormal: each of the
    sum's roundings is half of f32's least number there, over weights of 2^-8."""
    H, nKV, D = 4, 2, 64
    q, row_start, lens, tables, k, v = attention_case(46, dtype, H, nKV, D, P, [300, 64, 41], [3, 1, 2] if ragged else [1, 1, 1])
    v = R.stored(R.value(v, dtype) * 1e-36, dtype)
    got = run_attention(q, row_start, lens, tables, k, v, ragged, room=room).reshape(q.shape)
    want, mag, big = R.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype), R.value(v, dtype))
    rel = 2 * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) * big + 2.0 ** -20 + int(max(lens)) * 2.0 ** -23
    # three parts of a weight at the most, and a join of four waves
    assert np.all(np.abs(got.astype(np.float64) - want) <= mag * rel[..., None] + (3 * 300 + 4) * 2.0 ** -150 * 2.0 ** 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ragged,room,P", FORMS)
@pytest.mark.parametrize("how", ["queries", "scale"])
def test_keys_up_to_1e35(dtype, ragged, room, P, how):
    """Large keys against small queries, or against a small scale: every product
    and sum is inside f32."""
    H, nKV, D = 4, 2, 64
    q, row_start, lens, tables, k, v = attention_case(43, dtype, H, nKV, D, P, [300, 64, 41], [3, 1, 2] if ragged else [1, 1, 1])
    k = R.stored(R.value(k, dtype) * 1e35, dtype)
    q = np.copysign(1 + np.abs(q), q)
    scale = 0.125
    if how == "queries":
        q = (q * 1e-35).astype(np.float32)
    else:
        scale = 0.125e-35
    case = q, row_start, lens, tables, k, v
    check_attention(run_attention(*case, ragged=ragged, scale=scale, room=room), *case, dtype, np.float32(scale))


def junk_of(x, dtype):
    return {"f32": np.float32(x), "f16": np.float16(x),
            "bf16": np.uint16(np.float32(x).view(np.uint32) >> 16 | (0x40 if np.isnan(x) else 0))}[dtype]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("room", [0, room_for_many(4, 2, 2)])
@pytest.mark.parametrize("D,dim", [(64, 5), (72, 71), (128, 0)])
@pytest.mark.parametrize("where", ["key", "value"])
def test_one_entry_that_is_not_finite(dtype, room, D, dim, where):
    """Key 3 is seen by all rows, and lies in a tile that is; 150 too, in one beside
    hidden keys; 205 by the last rows only.  What the rows that see it may give is
    what the header says; the others, and other KV heads, are as without it."""
    H, nKV, P = 4, 2, 16
    q, row_start, lens, tables, k, v = attention_case(47, dtype, H, nKV, D, P, [210, 40], [60, 1])
    clean = run_attention(q, row_start, lens, tables, k, v, True, room=room).reshape(q.shape)
    near = lambda a, b: np.linalg.norm(a - b) <= 1e-5 * np.linalg.norm(b)
    pool = k if where == "key" else v
    for junk in (np.nan, np.inf, -np.inf):
        for at in (3, 150, 205):
            place = tables[0, at // P], 1, at % P, dim
            kept, pool[place] = pool[place], junk_of(junk, dtype)
            got = run_attention(q, row_start, lens, tables, k, v, True, room=room).reshape(q.shape)
            sees = np.zeros(q.shape[:2], bool)
            sees[:60, 2:] = (210 - 60 + np.arange(60) >= at)[:, None]
            assert near(got[~sees], clean[~sees]), (junk, at)
            if where == "value":
                assert not np.isfinite(got[sees][:, dim]).any(), (junk, at)
                for a, b in zip(np.delete(got[sees], dim, 1), np.delete(clean[sees], dim, 1)):
                    assert np.isnan(a).all() or near(a, b), (junk, at)
            elif np.isnan(junk):
                assert np.isnan(got[sees]).all(), (junk, at)
            else:
                with np.errstate(invalid="ignore"):
                    want, _, _ = R.attention(q.astype(np.float64), row_start, lens, tables, R.value(k, dtype),
                                             R.value(v, dtype))
                for a, w in zip(got[sees], want[sees]):  # a score of -inf weighs nothing
                    assert not np.isfinite(a).any() or (np.isfinite(w).all() and near(a, w)), (junk, at)
            pool[place] = kept
