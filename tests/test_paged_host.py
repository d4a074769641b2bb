"""PagedCache's bookkeeping on the host, on a device that is a dict: what it
allocates, gives back and moves, also where an allocation fails."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device

CONFIG = dict(maxSeqLen=64, numKVHeads=2, headDim=16, numLayers=3)


class FakeDevice:
    """Memory by address, a megabyte apart; calls that compute do nothing."""

    def __init__(self):
        self.memory, self.room, self.moved = {}, None, []

    def alloc(self, nbytes, mode=0):
        if self.room is not None:
            if not self.room:
                raise RuntimeError("out of memory")
            self.room -= 1
        self.last = getattr(self, "last", 0) + (1 << 20)
        self.memory[self.last] = np.zeros(int(nbytes), np.uint8)
        return self.last

    def release(self, address):
        del self.memory[address]

    def at(self, address, nbytes):
        base = address >> 20 << 20
        return self.memory[base][address - base:address - base + nbytes]

    def upload(self, address, a, offset=0):
        a = np.ascontiguousarray(a)
        self.moved.append(a.nbytes)
        self.at(address + offset, a.nbytes)[:] = np.frombuffer(a.tobytes(), np.uint8)

    def download(self, address, nbytes, dtype, offset=0):
        self.moved.append(nbytes)
        return self.at(address + offset, nbytes).copy().view(dtype)

    # of libsmith
    def smith_paged_plan(self, *a):
        return 0

    def smith_copy_d2d(self, ctx, dst, to, src, of, nbytes):
        self.at(dst + to, nbytes)[:] = self.at(src + of, nbytes)
        return 0

    def smith_set_i32(self, ctx, p, v):
        self.at(p, 4).view(np.int32)[0] = v
        return 0


@pytest.fixture
def fake(monkeypatch):
    f = FakeDevice()
    for name, what in (("alloc", f.alloc), ("release_buffer", f.release), ("upload", f.upload), ("download", f.download),
                       ("ops_ctx", lambda: None), ("lib", f)):
        monkeypatch.setattr(device, name, what)
    return f


def test_rows_that_there_is_no_memory_for(fake):
    """A larger pair of row buffers that cannot be had leaves the one there is."""
    cache = S.createPagedCache(CONFIG, 2, 2000, 16)
    cache.maxPages = 1000
    kept = cache.plan([3, 1])["slots"]
    before = cache.lens.copy(), cache.freeCount, dict(fake.memory)
    for room in (0, 1):
        fake.room = room
        with pytest.raises(RuntimeError, match="out of memory"):
            cache.plan([300, 0])
        assert cache.lens.tolist() == before[0].tolist() and cache.freeCount == before[1]
        assert fake.memory.keys() == before[2].keys()
    plan = cache.plan([0, 200])
    assert plan["slots"] is kept and kept.buffer
    fake.room = None
    plan = cache.plan([300, 0])
    assert plan["slots"].shape[0] >= 300 and plan["slots"].buffer and kept.buffer is None
    cache.free()
    assert not fake.memory


def test_a_cache_that_there_is_no_memory_for(fake):
    """Whichever allocation fails: what was had goes back."""
    for room in range(100):
        fake.room = room
        try:
            cache = S.createPagedCache(CONFIG, 3, 20, 16)
        except RuntimeError:
            assert not fake.memory, room
        else:
            break
    assert room == 14  # three layers' pools, tables, free list, two lengths and two counts, added, row starts
    cache.free()
    assert not fake.memory


def test_a_cache_that_was_freed(fake):
    """Nothing is done on memory that it no longer has."""
    cache = S.createPagedCache(CONFIG, 2, 20, 16)
    cache.plan([20, 3])
    cache.free()
    cache.free()
    for call in (lambda: cache.plan([1, 0]), lambda: cache.release(0), lambda: cache.append(0, {}, 0, 0, 1, 2, 0, 0, 0, 0),
                 lambda: cache.attention(0, {}, 0, 0, 1, 2, 0)):
        with pytest.raises(ValueError, match="paged cache: it was freed"):
            call()
    assert not fake.memory


@pytest.mark.parametrize("requests,pages", [(2, 40), (3000, 40000)])
def test_release_moves_one_requests_pages(fake, requests, pages):
    """However large the cache is: nothing is copied to the host, and the request's
    own pages on the device."""
    cache = S.createPagedCache(dict(CONFIG, numLayers=0, maxSeqLen=320), requests, pages, 16)
    added = np.zeros(requests, int)
    added[:2] = 33, 50
    cache.plan(added)
    tables = np.full((requests, 20), -1)
    tables[0, :3], tables[1, :4] = [7, 2, 30], [9, 0, 5, 31]  # as the step's kernel would
    cache._tables.set_data(tables)
    cache._lens[cache._turn].set_data(cache.lens)
    fake.moved.clear()
    cache.release(0)
    cache.release(0)
    assert sum(fake.moved) <= 64
    assert cache.freeCount == pages - 4 and cache.lens[:2].tolist() == [0, 50]
    assert cache._free.data[pages - 7:pages - 4].tolist() == [7, 2, 30]
    assert cache._count[cache._turn].data.tolist() == [pages - 4]
    assert cache._lens[cache._turn].data.tolist() == cache.lens.tolist()
    cache.release(1)
    assert cache._free.data[pages - 4:].tolist() == [9, 0, 5, 31] and cache.freeCount == pages
    with pytest.raises(ValueError, match="request %d of" % requests):
        cache.release(requests)
