"""What a step without a window asks of the host before its plan: nothing of each request."""
import numpy as np
import pytest

import smith_amd as S
from test_paged_fork_host import check, fake  # noqa: F401
from test_paged_host import CONFIG


def test_room_without_a_window_asks_nothing_of_the_requests(fake, monkeypatch):
    cache = S.createPagedCache(CONFIG, 3, 8, 4)
    cache.plan([5, 0, 9])

    def asked(*a):
        raise AssertionError("a request was looked at")
    monkeypatch.setattr(cache, "_pages", asked)
    monkeypatch.setattr(cache, "trim", asked)
    cache.make_room([1, 30, 1])  # 8 new pages, 3 are free: the plan says so
    with pytest.raises(ValueError, match="paged step: 8 new pages, 3 are free"):
        cache.plan([1, 30, 1])


@pytest.mark.parametrize("free,trims", [(2, False), (1, True)])
def test_room_with_a_window(fake, monkeypatch, free, trims):
    """Pages are given back only if the step's rows need more than are free."""
    cache = S.createPagedCache(CONFIG, 3, 10 + free, 4, window=8)
    cache.plan([30, 0, 7])  # 8 and 2 pages; of the first 22 .. 29 are seen, pages 5 .. 7
    calls, trim = [], cache.trim
    monkeypatch.setattr(cache, "trim", lambda: calls.append(trim()))
    cache.make_room([2, 4, 2])  # page 0 of request 1, page 2 of request 2
    assert bool(calls) == trims and cache.freeCount == (7 - 1 if trims else 2)
    cache.plan(np.array([2, 4, 2]))
    check(cache)
