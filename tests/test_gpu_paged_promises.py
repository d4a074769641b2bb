"""Statements of include/smith.h that no other test makes true: several rows that are wrong
at once, and the page of the next key under the smallest window."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import pages_reference as P_
import paged_reference as R
from test_gpu_paged import i32, last_error
from test_gpu_paged_fork import moved, pools_of, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [300, 60000])
def test_of_several_rows_with_a_token_outside_one_is_named(vocab):
    x = np.random.RandomState(1).standard_normal((40, vocab)).astype(np.float32)
    tokens = np.full((40, 2), 7, np.int32)
    wrong = [3, 17, 39]
    tokens[wrong, 1] = vocab
    r = S.logProbs(R.upload(x), R.upload(tokens))
    assert device.lib.smith_sync(device.ctx()) == -1
    assert last_error() in ["smith_logprobs: row %d: a token outside the vocabulary" % b for b in wrong]
    device.sync()
    assert np.array_equal(np.isnan(r["logprobs"].data), tokens == vocab)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("P", [4, 16])
def test_compact_keeps_the_page_of_the_next_key(P, dtype):
    """A window of one key sees none of those that are there: a partly filled page stays."""
    rs, lens, tables, n_pages = state(P, 30, P, 90, 20)
    pools = pools_of(rs, 3, n_pages, 2, P, 8, dtype)
    want = P_.compact(lens, tables, n_pages, P, np.zeros(n_pages, np.int32), 1, 0)
    dev, t = [R.upload(p) for p in pools], i32(tables)
    new = S.pagedCompact(i32(lens), t, dev, 1, 0)
    device.sync()
    got = t.data
    for b, n in enumerate(lens):
        for j in range(-(-int(n) // P)):
            assert got[b, j] == want[0][b, j]
            assert (got[b, j] >= 0) == (j == n // P)
    count = new["freeCount"].data[0]
    assert count == want[2] and np.array_equal(new["freePages"].data[:count], want[1][:count])
    for t, x in zip(dev, moved(pools, [(a, b, P) for a, b in want[3]])):
        live = [int(got[b, n // P]) for b, n in enumerate(lens) if n % P]
        assert np.array_equal(t.data[live], x[live])
