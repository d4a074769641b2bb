"""Steps of a paged cache that fail half way, and caches that do."""
import numpy as np
import pytest

from smith_amd import device, paged
from smith_amd import tensor as T
from smith_amd.gguf_loader import loadGGUF
from llama_fixtures import write_tiny_llama

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def path(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("gguf") / "q4.gguf")
    write_tiny_llama(p, dim=256, layers=2, heads=4, kv_heads=2, ffn=512, vocab=320, context=1024)
    return p


@pytest.fixture(scope="module")
def model(path):
    return loadGGUF(path)


FIRST, SECOND = [[3, 77, 150, 9], [5], [8] * 20], [[1, 2, 3], [250] * 17, []]


class Failure(Exception):
    pass


@pytest.mark.parametrize("where", ["append", "attention", "download", "interrupt"])
def test_a_step_that_fails_can_be_repeated(model, monkeypatch, where):
    """Whatever raises, and wherever: the cache is as it was before the step."""
    want, cache = [], model.createPagedCache(3, 40, 4, "f32")
    for tokens in (FIRST, SECOND, FIRST):
        want.append(model.forwardPagedStep(tokens, cache)["logits"])
    cache.free()
    cache = model.createPagedCache(3, 40, 4, "f32")
    for tokens, w in zip((FIRST, SECOND, FIRST), want):
        before = cache.lens.copy(), cache.freeCount
        with monkeypatch.context() as m:
            if where == "download":
                def fail(*a, **k):
                    raise Failure
                m.setattr(device, "download_into", fail)
            else:
                name = "append" if where == "append" else "attention"
                run = getattr(paged.PagedCache, name)

                def fail(self, layer, *a):
                    if layer == 1:
                        raise KeyboardInterrupt if where == "interrupt" else Failure
                    run(self, layer, *a)
                m.setattr(paged.PagedCache, name, fail)
            with pytest.raises((Failure, KeyboardInterrupt)):
                model.forwardPagedStep(tokens, cache)
        assert np.array_equal(cache.lens, before[0]) and cache.freeCount == before[1]
        assert np.array_equal(model.forwardPagedStep(tokens, cache)["logits"], w)
    cache.release(1)  # a request that a failed step had grown gives back what it has
    assert cache.freeCount == 40 - sum(-(-int(n) // 4) for n in cache.lens)
    cache.free()


def test_no_memory_for_the_logits(path, monkeypatch):
    """Found out before the step begins."""
    model = loadGGUF(path)
    cache = model.createPagedCache(3, 40, 4, "f32")
    planned = []
    with monkeypatch.context() as m:
        from smith_amd import gguf_cache

        def fail(self):
            raise Failure
        m.setattr(gguf_cache._Engine, "_row_logits", fail)
        m.setattr(paged.PagedCache, "plan", lambda self, added: planned.append(added))
        with pytest.raises(Failure):
            model.forwardPagedStep(FIRST, cache)
    assert not planned and model.forwardPagedStep(FIRST, cache)["logits"].shape == (3, 320)
    cache.free()
