"""The bars for the norm of attention's errors tell a part of q or of the weights that is
lost from all of them: on the CPU, at the sizes of the tests on the device."""
import numpy as np
import pytest

import accuracy_reference as A


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("keys", [40, 300, 1500])
@pytest.mark.parametrize("dtype,terms", [("f16", 2), ("bf16", 3)])
@pytest.mark.parametrize("q_std", list(A.BARS))
def test_a_lost_part_is_seen(D, keys, dtype, terms, q_std):
    rs = np.random.RandomState(D + keys)
    q = (rs.standard_normal((60, D)) * q_std).astype(np.float32).astype(np.float64)
    k, v = (A.parts(rs.standard_normal((keys, D)), dtype, 1) for _ in range(2))
    want = A.attention(q, k, v)
    A.check_norm(A.attention(q, k, v, dtype, terms, terms), want, [keys] * 60, q_std)
    lost = (terms - 1, terms) if q_std == 2 else (terms, terms - 1)
    with pytest.raises(AssertionError):
        A.check_norm(A.attention(q, k, v, dtype, *lost), want, [keys] * 60, q_std)
