"""A free list that is shorter than its count says."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
from test_gpu_paged import i32, sync_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [5, 20, 24])
def test_count_past_the_list(count):
    """No page is read from behind a list of smith_alloc's memory."""
    cached, tables = np.array([5, 16], np.int32), np.arange(8, dtype=np.int32).reshape(2, 4)
    t = i32(tables)
    plan = S.pagedPlan(i32(cached), i32([1, 3]), i32([20, 21, 22, 23]), i32([count]), t, 24, 16, 10)
    assert "the %d free pages, or the list holds fewer" % count in sync_error()
    assert np.array_equal(t.data, tables) and np.array_equal(plan["lens"].data, cached)
    assert not plan["rowStart"].data.any() and (plan["slots"].data == -1).all() and plan["freeLeft"].data[0] == count


def test_whole_list():
    t = i32(np.arange(8, dtype=np.int32).reshape(2, 4))
    plan = S.pagedPlan(i32([5, 16]), i32([1, 3]), i32([20, 21, 22, 23]), i32([4]), t, 24, 16, 10)
    device.sync()
    assert t.data[1].tolist() == [4, 23, 6, 7] and plan["freeLeft"].data[0] == 3
