"""Continuations, windows and scores of a loaded GGUF model, run together as a server
would: against the same model's requests alone."""
import numpy as np
import pytest

from smith_amd import device, paged
from smith_amd.gguf_loader import loadGGUF
from llama_fixtures import write_tiny_llama
from test_gpu_paged_llama import BAR, Alone, off

pytestmark = pytest.mark.gpu
SMALL = dict(dim=256, layers=2, heads=4, kv_heads=2, ffn=512, vocab=320, context=2048)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("gguf") / "q4.gguf")
    write_tiny_llama(p, **SMALL)
    return loadGGUF(p)


def log_softmax(x):
    x = x.astype(np.float64)
    return x - x.max(1, keepdims=True) - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True))


class Texts:
    """What each request has been given, and the model's logits behind it alone."""

    def __init__(self, model, n):
        self.m, self.texts = model, [[] for _ in range(n)]

    def step(self, tokens):
        out = []
        for text, t in zip(self.texts, tokens):
            text += t
            if t:
                out.append(self.m.forwardPrefill(text, self.m.createCache())["logits"][-1])
        return np.stack(out)

    def fork(self, parents):
        self.texts = [list(self.texts[p]) if p >= 0 else [] for p in parents]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("apart", [False, True])
def test_continuations(model, dtype, page, apart, monkeypatch):
    """A prompt that goes on in several ways, beams that go on from others, requests
    that end, the pool made smaller and larger; with the shared keys read by each
    request, and once for all."""
    if apart:
        monkeypatch.setattr(paged, "SHARED_BYTES", 1)
    n = 6
    cache, alone = model.createPagedCache(n, 200, page, dtype), Texts(model, n)
    rs = np.random.RandomState(page)

    def step(tokens):
        r = model.forwardPagedStep(tokens, cache)
        want = alone.step(tokens)
        assert (off(r["logits"], want) <= BAR[dtype]).all(), off(r["logits"], want)

    def fork(parents):
        cache.fork(parents)
        alone.fork(parents)
    device.profile_kernels(True)
    try:
        step([rs.randint(0, 320, 37).tolist(), [], [], rs.randint(0, 320, 16).tolist(), [], []])
        fork([0, 0, 0, 3, 3, -1])
        step([[1], [2], [3], [4], [5], [6, 7, 8]])
        step([[9], [10, 11], [12], [13], [], [14]])
        fork([2, 0, 0, 4, 4, 5])
        step([[15], [16], [17, 18, 19], [20], [21], [22]])
        cache.release(1)
        alone.fork([0, -1, 2, 3, 4, 5])
        live = cache.compact()
        assert live == cache.pages - cache.freeCount
        step([[23], rs.randint(0, 320, 20).tolist(), [24], [25], [26], [27]])
        cache.resize(cache.compact() + 12)
        step([[28], [29], [30], [31], [32], [33]])
        cache.resize(100)
        fork([3, 3, 3, 3, 0, 0])
        step([[34], [35], [36], [37], [38], [39]])
        shared = device.profile_read("smith_paged_attention_own")[1]
        assert bool(shared) == apart
    finally:
        device.profile_kernels(False)
        device.profile_read("")
    assert cache.lens.tolist() == [len(t) for t in alone.texts]
    for b in range(n):
        cache.release(b)
    assert cache.freeCount == cache.pages == 100
    cache.free()


def test_equal_continuations_have_equal_logits(model):
    """Beams from one parent are the same request until they are given other tokens."""
    cache = model.createPagedCache(4, 60, 8, "f16")
    model.forwardPagedStep([[5, 6, 7, 8, 9, 10, 11, 12, 13, 14], [], [], []], cache)
    cache.fork([0, 0, 0, 0])
    r = model.forwardPagedStep([[3]] * 4, cache)["logits"]
    assert np.array_equal(r, np.broadcast_to(r[0], r.shape))
    cache.free()


def test_a_step_that_fails_after_a_fork(model, monkeypatch):
    cache = model.createPagedCache(3, 40, 4, "f32")
    model.forwardPagedStep([[1, 2, 3, 4, 5, 6], [], [7]], cache)
    cache.fork([0, 0, 2])
    before = cache.lens.tolist(), cache.freeCount
    with monkeypatch.context() as m:
        def fail(*a, **k):
            raise RuntimeError("no")
        m.setattr(device, "download_into", fail)
        with pytest.raises(RuntimeError, match="no"):
            model.forwardPagedStep([[8, 9, 10, 11], [12], []], cache)
    assert (cache.lens.tolist(), cache.freeCount) == before
    got = model.forwardPagedStep([[8, 9, 10, 11], [12], []], cache)["logits"]
    alone = Texts(model, 2)
    alone.texts = [[1, 2, 3, 4, 5, 6], [1, 2, 3, 4, 5, 6]]
    assert (off(got, alone.step([[8, 9, 10, 11], [12]])) <= BAR["f32"]).all()
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_long_chat_in_few_pages(model, dtype):
    """With a window a chat goes on for longer than its pages could hold, and what it is
    given back serves another; the logits are those of a cache that keeps everything."""
    window, sinks, P = 24, 3, 4
    few, all_ = (model.createPagedCache(2, pages, P, dtype, window, sinks) for pages in (18, 400))
    rs = np.random.RandomState(0)
    text = rs.randint(0, 320, 150).tolist()
    at, turn = 0, 0
    while at < 150:
        k = [1, 9, 1, 4][turn % 4]
        step = [text[at:at + k], [int(rs.randint(320))] if turn % 3 else []]
        a, b = model.forwardPagedStep(step, few), model.forwardPagedStep(step, all_)
        assert (off(a["logits"], b["logits"]) <= 1e-5).all()
        at, turn = at + k, turn + 1
    assert few.lens.tolist() == all_.lens.tolist() and few.lens[0] == 150
    few.trim()
    assert few.freeCount == 18 - sum(len([x for x in ids if x is not None]) for ids in few._ids)
    assert few.freeCount >= 18 - 2 * (1 + -(-window // P) + 1) - 1
    # a window that sees everything is no window
    whole, plain = model.createPagedCache(1, 60, P, dtype, 500), model.createPagedCache(1, 60, P, dtype)
    for t in (text[:40], text[40:41], text[41:50]):
        a, b = (model.forwardPagedStep([t], c)["logits"] for c in (whole, plain))
        assert (off(a, b) <= 1e-5).all()
    for c in (few, all_, whole, plain):
        c.free()


def test_scores_of_a_text(model):
    """score() is the log softmax of the prompt's logits, as the host would work it out."""
    text = np.random.RandomState(1).randint(0, 320, 300).tolist()
    lg = log_softmax(model.forwardPrefill(text[:-1], model.createCache())["logits"])
    r = model.score(text, 7)
    want = lg[np.arange(299), text[1:]]
    # the same logits; a number of these is off by a few half steps of its terms (at most 2^-20 of 10)
    assert np.abs(r["logprobs"] - want).max() <= 1e-5
    assert np.abs(r["entropy"] + (np.exp(lg) * lg).sum(1)).max() <= 1e-5
    assert np.array_equal(r["topIds"], np.argsort(-lg, 1, kind="stable")[:, :7])
    assert np.abs(r["topLogprobs"] - np.sort(lg, 1)[:, ::-1][:, :7]).max() <= 1e-5
    assert model.score(text[:2])["logprobs"].shape == (1,) and model.score(text[:2])["topIds"].shape == (1, 0)
    for bad, top, message in (([1], 0, "a text of 1"), ([1, 320], 0, "outside the vocabulary"), ([1, 2], 65, "65 top"),
                              ([1, 2], -1, "-1 top")):
        with pytest.raises(ValueError, match="score: .*" + message):
            model.score(bad, top)


def test_score_gives_its_memory_back(model):
    text = list(range(40))
    model.score(text, 3)
    before = device.allocated_size()
    model.score(text, 3)
    assert device.allocated_size() == before


def test_beam_search(model):
    """Two beams over scored steps against all of their continuations one by one: the
    score of a beam is the sum of its tokens' log probabilities."""
    prompt, width = [3, 77, 150, 9, 210, 44, 1], 3
    cache = model.createPagedCache(width, 60, 4, "f32")
    r = model.scorePagedStep([prompt] + [[]] * (width - 1), cache, width)
    assert r["requests"] == [0] and r["topIds"].shape == (1, width) and r["entropy"].shape == (1,)
    cache.fork([0] * width)
    texts = [prompt + [int(t)] for t in r["topIds"][0]]
    scores = r["topLogprobs"][0].astype(np.float64)
    for _ in range(6):
        r = model.scorePagedStep([t[-1:] for t in texts], cache, width)
        total = scores[:, None] + r["topLogprobs"]
        best = np.argsort(-total.ravel(), kind="stable")[:width]
        parents = best // width
        texts = [texts[p] + [int(r["topIds"][p, i % width])] for p, i in zip(parents, best)]
        scores = total.ravel()[best]
        cache.fork(parents)
    for t, s in zip(texts, scores):
        want = model.score(t)["logprobs"][len(prompt) - 1:].astype(np.float64).sum()
        # 7 tokens' log probabilities, whose logits (of a few units) differ by BAR between the two ways
        assert abs(want - s) <= 7 * 2 * BAR["f32"] * 8
    with pytest.raises(ValueError, match="0 top"):
        model.scorePagedStep([[1]] * width, cache, 0)
    cache.free()
