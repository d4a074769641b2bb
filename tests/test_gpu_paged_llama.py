"""forwardPagedStep of a loaded GGUF model against the same model's cache of one
request: several requests in one step, of any lengths, on a shared pool."""
import numpy as np
import pytest

from smith_amd import createPagedCache, device
from smith_amd.gguf_loader import loadGGUF
from llama_fixtures import write_tiny_llama

pytestmark = pytest.mark.gpu

SMALL = dict(dim=256, layers=2, heads=4, kv_heads=2, ffn=512, vocab=320, context=1024)
# The two ways run the same products on other numbers of rows, and a product of
# several rows rounds its activations to f16 (half a step: 2^-11) where one of a
# single row does not: 4 products in each of 2 layers, so 8 * 2^-11 of the norm at
# most.  The cache's rounding of keys and of values adds half a step of its type each.
BAR = {t: 8 * 2.0 ** -11 + 2 * half for t, half in (("f32", 0.0), ("f16", 2.0 ** -11), ("bf16", 2.0 ** -8))}


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("gguf") / "q4.gguf")
    write_tiny_llama(p, **SMALL)
    return loadGGUF(p)


class Alone:
    """Each request on a cache of its own."""

    def __init__(self, model, n):
        self.m, self.caches, self.len = model, [model.createCache() for _ in range(n)], [0] * n

    def step(self, tokens):
        out = []
        for b, t in enumerate(tokens):
            if not t:
                continue
            if self.len[b] == 0:
                lg = self.m.forwardPrefill(t, self.caches[b])["logits"][-1]
            else:
                for i, x in enumerate(t):
                    lg = self.m.forwardDecode(x, self.len[b] + i, self.caches[b])["logits"][0]
            self.len[b] += len(t)
            out.append(lg)
        return np.stack(out)


def off(got, want):
    return np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)


STEPS = [[[3, 77, 150, 9, 210, 44, 1], [5], [], [8, 8, 8, 9]],      # prompts
         [[5], [250, 17, 31, 4, 2, 6], [99, 100], [7]],             # decode rows, a chunk, a late prompt
         [[1], [], [2], [3]], [[4], [5], [6], [7]],
         [[10, 20, 30], [40], [50, 60, 70, 80, 90], []], [[11], [12], [13], [14]]]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [4, 16])
def test_steps_match_requests_alone(model, dtype, page):
    cache = model.createPagedCache(4, 64, page, dtype)
    alone = Alone(model, 4)
    for i, tokens in enumerate(STEPS):
        r = model.forwardPagedStep(tokens, cache)
        want = alone.step(tokens)
        assert r["requests"] == [b for b in range(4) if tokens[b]]
        assert r["logits"].shape == want.shape
        assert (off(r["logits"], want) <= BAR[dtype]).all(), (i, off(r["logits"], want))
    assert cache.lens.tolist() == alone.len


def test_greedy_requests_together_and_alone(model):
    """Three requests decoded together, fed with what generate gives each alone:
    generate's token is the best there too, or as good within the bar."""
    prompts = [[3, 77, 150], [9], [210, 44, 1, 250, 17]]
    alone = [model.generate(p, {"maxTokens": 12, "temperature": 0})[len(p):] for p in prompts]
    cache = model.createPagedCache(3, 40, 8, "f32")
    feed, same = prompts, 0
    for i in range(12):
        for lg, tokens in zip(model.forwardPagedStep(feed, cache)["logits"], alone):
            assert lg[tokens[i]] >= lg.max() - 2 * BAR["f32"] * np.abs(lg).max()
            same += int(lg.argmax()) == tokens[i]
        feed = [[t[i]] for t in alone]
    assert same >= 30  # of 36


def test_pages_are_given_back_and_taken_again(model):
    """A request's pages serve others after it, in another order; the results are
    those of a fresh cache, and the pool never grows."""
    cache = model.createPagedCache(3, 6, 4, "f32")
    alone = Alone(model, 3)
    first = [[1, 2, 3, 4, 5], [6, 7, 8, 9], [10, 11, 12]]
    model.forwardPagedStep(first, cache)
    alone.step(first)
    assert cache.freeCount == 2
    with pytest.raises(ValueError, match="3 new pages, 2 are free"):
        model.forwardPagedStep([[1] * 4, [2], [3, 4]], cache)
    assert cache.lens.tolist() == [5, 4, 3] and cache.freeCount == 2  # nothing happened
    cache.release(0)
    assert cache.freeCount == 4
    cache.release(0)  # of a request without pages: nothing
    assert cache.freeCount == 4
    alone.caches[0], alone.len[0] = model.createCache(), 0
    for tokens in ([[20, 21, 22], [13, 14], [15]], [[23, 24], [], [16, 17]], [[25], [18, 19], []]):
        r = model.forwardPagedStep(tokens, cache)
        want = alone.step(tokens)
        assert (off(r["logits"], want) <= BAR["f32"]).all()
    assert cache.freeCount == 6 - sum(-(-int(n) // 4) for n in cache.lens)


def test_refusals(model):
    cache = model.createPagedCache(2, 200, 16, "f16")
    with pytest.raises(ValueError, match="tokens of 3 requests"):
        model.forwardPagedStep([[1], [2], [3]], cache)
    with pytest.raises(ValueError, match="one at least"):
        model.forwardPagedStep([[], []], cache)
    with pytest.raises(ValueError, match="257 rows"):
        model.forwardPagedStep([[1] * 200, [2] * 57], cache)
    with pytest.raises(ValueError, match="whole-row RoPE"):
        model.forwardPagedStep([[1] * 256, []], cache) and model.forwardPagedStep([[1], []], cache)
    with pytest.raises(ValueError, match="outside the vocabulary"):
        model.forwardPagedStep([[], [3, 320]], cache)
    with pytest.raises(ValueError, match="outside the vocabulary"):
        model.forwardPagedStep([[], [-1]], cache)
    for b in (-1, 2):
        with pytest.raises(ValueError, match="request %d of 2" % b):
            cache.release(b)
    other = createPagedCache(dict(model.model["config"], numLayers=1), 2, 10)
    with pytest.raises(ValueError, match="a cache of 1 layers"):
        model.forwardPagedStep([[1], [2]], other)
    assert cache.lens.tolist() == [256, 0] and cache.freeCount == 184 and other.freeCount == 10
    with pytest.raises(ValueError, match="pages of q8"):
        model.createPagedCache(2, 10, 16, "q8")
    with pytest.raises(ValueError, match="power of two"):
        model.createPagedCache(2, 10, 12)
    with pytest.raises(ValueError, match="0 requests"):
        model.createPagedCache(0, 10)


def test_a_cache_gives_its_memory_back(model):
    before = device.allocated_size()
    cache = model.createPagedCache(2, 64, 16, "f16")
    model.forwardPagedStep([[1, 2], [3]], cache)
    grown = device.allocated_size()  # with what the model keeps for such steps
    cache.free()
    model_keeps = device.allocated_size() - before
    again = model.createPagedCache(2, 64, 16, "f16")
    model.forwardPagedStep([[1, 2], [3]], again)
    assert device.allocated_size() - before - model_keeps == grown - before - model_keeps > 0
    again.free()
    assert device.allocated_size() - before == model_keeps
    with pytest.raises(ValueError, match="a cache of 0 layers"):
        model.forwardPagedStep([[1], [2]], cache)


def test_many_rows_in_one_step(model):
    """256 rows of prompts."""
    rs = np.random.RandomState(3)
    tokens = [rs.randint(0, 320, n).tolist() for n in (100, 1, 60, 95)]
    cache = model.createPagedCache(4, 20, 16, "f16")
    got = model.forwardPagedStep(tokens, cache)["logits"]
    assert (off(got, Alone(model, 4).step(tokens)) <= BAR["f16"]).all()
