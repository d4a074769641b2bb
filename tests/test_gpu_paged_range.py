"""Paged attention where weights, keys or values span far: what f32 arithmetic
holds of them is held, and what f16 pages lose is no more than is stated."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import attention_case, check_attention, room_for_many, run_attention

pytestmark = pytest.mark.gpu

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
