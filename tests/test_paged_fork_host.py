"""PagedCache's bookkeeping of shared pages on the host, on a device that is a dict and
calls that are the plain forms: what it counts is what the device's tables and lists say."""
import ctypes

import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import pages_reference as P_
import paged_reference as R
from test_paged_host import CONFIG, FakeDevice


class Device(FakeDevice):
    """Plan, fork and compact as the references do them; `shared`: the last shared attention."""
    shared = None

    def ints(self, address, n):
        return self.at(address, 4 * n).view(np.int32)

    def smith_paged_plan(self, ctx, cached, added, n, free, count, n_pages, P, max_pages, max_rows, tables, row_start, lens,
                         slots, positions, left):
        t = self.ints(tables, n * max_pages).reshape(n, max_pages)
        c, a = self.ints(cached, n), self.ints(added, n)
        r = R.plan(c, a, self.ints(free, n_pages), self.ints(count, 1)[0], t, P, max_rows)
        t[:] = r[0]
        self.ints(row_start, n + 1)[:], self.ints(lens, n)[:] = r[1], r[2]
        self.ints(left, 1)[0] = r[5]
        return 0

    def smith_paged_fork(self, ctx, kv, lens, tables, parents, n, max_pages, window, sinks, nKV, hd, pools, n_pools, n_pages, P,
                         new_lens, new_tables, free, count):
        assert n_pools == len(pools)
        t = self.ints(new_tables, n * max_pages).reshape(n, max_pages)
        f = self.ints(free, n_pages)
        r = P_.fork(self.ints(lens, n).copy(), self.ints(tables, n * max_pages).reshape(n, max_pages), self.ints(parents, n),
                    n_pages, P, t, f, window, sinks)
        self.ints(new_lens, n)[:], t[:], f[:] = r[0], r[1], r[2]
        self.ints(count, 1)[0] = r[3]
        return 0

    def smith_paged_compact(self, ctx, kv, lens, tables, n, max_pages, window, sinks, nKV, hd, pools, n_pools, n_pages, P,
                            new_tables, free, count):
        t = self.ints(tables, n * max_pages).reshape(n, max_pages)
        f = self.ints(free, n_pages)
        r = P_.compact(self.ints(lens, n), t, n_pages, P, f, window, sinks)
        self.ints(new_tables, n * max_pages)[:], f[:] = r[0].ravel(), r[1]
        self.ints(count, 1)[0] = r[2]
        return 0

    def smith_paged_attention(self, *a):
        self.shared = None
        return 0

    def smith_paged_attention_shared(self, *a):
        self.shared = a
        return 0

    def smith_paged_attention_window(self, *a):
        self.window = a[10], a[11]
        return 0


@pytest.fixture
def fake(monkeypatch):
    f = Device()
    for name, what in (("alloc", f.alloc), ("release_buffer", f.release), ("upload", f.upload), ("download", f.download),
                       ("ops_ctx", lambda: None), ("lib", f), ("sync", lambda: None)):
        monkeypatch.setattr(device, name, what)
    return f


def check(cache):
    """The device's side: every page in nobody's table or list once, the counts the same."""
    a = cache._turn
    assert cache._lens[a].data.tolist() == cache.lens.tolist()
    assert cache._count[a].data[0] == cache.freeCount
    tables, P, named = cache._tables.data, cache.pageSize, set()
    for b, n in enumerate(cache.lens):
        for j in range(-(-int(n) // P)):
            ids = cache._ids[b] if cache._ids is not None else None
            if ids is None or ids[j] is not None:
                named.add(int(tables[b, j]))
                if n % P and j == n // P and ids is not None:  # a partly filled page is its request's own
                    assert cache._named[ids[j]] == 1
    free = cache._free.data[:cache.freeCount].tolist()
    assert len(set(free)) == len(free) and not named & set(free)
    assert named | set(free) == set(range(cache.pages))
    for first, behind, pages in cache._groups:
        for b in range(first, behind):
            assert (tables[b, :pages] == tables[first, :pages]).all() and cache.lens[b] >= pages * P


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 0), (13, 6)])
@pytest.mark.parametrize("seed", range(6))
def test_any_sequence_of_calls(fake, seed, window, sinks):
    rs = np.random.RandomState(seed)
    n, P = 7, 4
    cache = S.createPagedCache(dict(CONFIG, numLayers=2, maxSeqLen=120), n, 60, P, "f16", window, sinks)
    for _ in range(120):
        what = rs.randint(8)
        try:
            if what < 3:
                added = rs.randint(0, 8, n) * (rs.rand(n) < 0.6)
                before = cache.state()
                cache.make_room(added)
                before = cache.state()
                cache.plan(added)
                if rs.rand() < 0.2:  # the step fails
                    cache.restore(before)
                    cache.plan(added)
            elif what < 5:
                cache.fork(np.where(rs.rand(n) < 0.6, np.arange(n), rs.randint(-1, n, n)))
            elif what == 5:
                cache.release(rs.randint(n))
            elif what == 6:
                assert cache.compact() == cache.pages - cache.freeCount
                assert set(cache._free.data[:cache.freeCount]) == set(range(cache.pages - cache.freeCount, cache.pages))
            elif rs.rand() < 0.3:
                cache.resize(int(cache.pages - cache.freeCount + rs.randint(1, 40)))
            elif window:
                cache.trim()
        except ValueError as e:
            assert "pages" in str(e) or "grows past" in str(e) or "one at least" in str(e), e
            if "grows past" in str(e):
                cache.release(int(cache.lens.argmax()))
        check(cache)
    cache.free()
    assert not fake.memory


def test_groups_and_which_attention_runs(fake, monkeypatch):
    from smith_amd import paged
    cache = S.createPagedCache(dict(CONFIG, maxSeqLen=400), 6, 100, 4)
    cache.plan([41, 0, 0, 9, 0, 0])
    cache.fork([0, 0, 0, 3, 3, -1])
    assert cache._groups == [[0, 3, 10], [3, 5, 2], [5, 6, 0]]
    assert cache.lens.tolist() == [41, 41, 41, 9, 9, 0] and cache.freeCount == 100 - 11 - 2 - 3 - 1
    assert cache._group_tensors[0].data.tolist() == [0, 3, 5, 6, 6, 6, 6]
    assert cache._group_tensors[1].data.tolist()[:3] == [40, 8, 0]
    plan = cache.plan([1, 1, 1, 1, 1, 1])
    cache.attention(0, plan, 0, 32, 6, 2, 0)
    assert fake.shared is None  # not worth it
    saved = 2 * 2 * 16 * 2 * (2 * 40 + 8)
    for bar, runs in ((saved, True), (saved + 1, False)):
        monkeypatch.setattr(paged, "SHARED_BYTES", bar)
        cache.attention(0, plan, 0, 32, 6, 2, 0)
        assert (fake.shared is not None) == runs
    assert cache._groups[2] == [5, 6, 0]
    cache.release(1)  # a request between others that ends ends their group
    assert cache._groups == [[0, 1, 0], [1, 2, 0], [2, 3, 0], [3, 5, 2], [5, 6, 0]]
    cache.plan([0, 30, 0, 0, 0, 0])
    check(cache)


def test_a_window_is_handed_on(fake):
    cache = S.createPagedCache(CONFIG, 2, 20, 4, window=10, sinks=3)
    plan = cache.plan([30, 2])
    cache.attention(0, plan, 0, 32, 32, 2, 0)
    assert fake.window == (10, 3)
    cache.trim()  # of 30 keys 0 .. 2 and 21 .. 29 are seen: pages 0 and 5 .. 7
    assert cache.freeCount == 20 - 4 - 1 and cache._ids[0][1:5] == [None] * 4
    cache.fork([0, 0])
    assert cache._groups == [] and cache.freeCount == 20 - 4 - 1
    check(cache)


def test_refusals(fake):
    cache = S.createPagedCache(CONFIG, 3, 6, 4)
    cache.plan([13, 5, 0])
    for bad in ([0, 1], [0, 1, 3], [-2, 0, 1], [0.0, 1.0, 2.0]):
        with pytest.raises(ValueError, match="parents are 3 numbers"):
            cache.fork(bad)
    with pytest.raises(ValueError, match="paged fork: 7 pages, there are 6"):
        cache.fork([0, 1, 0])
    assert cache.lens.tolist() == [13, 5, 0] and cache.freeCount == 0
    check(cache)
    with pytest.raises(ValueError, match="paged cache: 2 pages for the"):
        cache.resize(2)
    check(cache)
    for bad in ((-1, 0), (0, 3), (4, -1)):
        with pytest.raises(ValueError, match="a window of"):
            S.createPagedCache(CONFIG, 3, 6, 4, window=bad[0], sinks=bad[1])
    cache.free()
    for call in (lambda: cache.fork([0, 1, 2]), cache.trim, cache.compact, lambda: cache.resize(9)):
        with pytest.raises(ValueError, match="paged cache: it was freed"):
            call()
    assert not fake.memory


def test_no_memory(fake):
    """A fork, and a resize, that there is no memory for: nothing happens."""
    cache = S.createPagedCache(CONFIG, 2, 20, 4)
    cache.plan([9, 5])
    # tables, free list, parents, groups; three layers' pools and two free lists
    for call, most in ((lambda: cache.fork([0, 0]), 5), (lambda: cache.resize(8), 8)):
        for room in range(most):
            before, memory = cache.lens.tolist(), len(fake.memory)
            fake.room = room
            with pytest.raises(RuntimeError, match="out of memory"):
                call()
            assert cache.lens.tolist() == before and len(fake.memory) == memory
            fake.room = None
            check(cache)
        fake.room = most
        call()
        fake.room = None
        check(cache)
    cache.free()
    assert not fake.memory
