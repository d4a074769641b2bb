"""What an onToken callback may do with the model that is generating: score texts,
and step requests and prompts on caches of its own.  The generated text is the
same, and so are the scores."""
import numpy as np
import pytest

from smith_amd import gguf_cache
from smith_amd.gguf_loader import loadGGUF
from llama_fixtures import write_tiny_llama

pytestmark = pytest.mark.gpu
MODELS = {
    # a position is up to context / heads: rows of heads of 64 by the attention that
    # leaves partials, by rows that are no blocks of 32, and by the f32 head and heads of 16
    "q4_0": dict(dim=256, layers=2, heads=4, kv_heads=2, ffn=512, vocab=320, context=4096),
    "q8_0": dict(dim=256, layers=2, heads=4, kv_heads=2, ffn=512, vocab=320, context=4096, linear_type="q8_0"),
    "tied": dict(context=4096, tie=True),
}
PROMPT = [3, 77, 51, 9, 21, 44, 1]
WAYS = {"greedy": dict(temperature=0, maxTokens=24), "sampled": dict(temperature=0.9, seed=5, maxTokens=24),
        "penalty": dict(temperature=0, repetitionPenalty=1.3, maxTokens=24)}


@pytest.fixture(scope="module", params=list(MODELS))
def model(request, tmp_path_factory):
    p = str(tmp_path_factory.mktemp("gguf") / "m.gguf")
    write_tiny_llama(p, **MODELS[request.param])
    return loadGGUF(p)


def other_texts(vocab):
    """Of one row, of a few, of several chunks: longer and shorter than what is generated."""
    rs = np.random.RandomState(7)
    return [rs.randint(0, vocab, n).tolist() for n in (2, 3, 40, 300, 12, 600)]


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("graph", [True, False])
def test_scores_of_other_texts(model, way, graph, monkeypatch):
    monkeypatch.setattr(gguf_cache, "USE_GRAPH", graph)
    alone, got, scores = [], [], []
    texts = other_texts(model.config["vocabSize"])
    want = [model.score(t, 3) for t in texts]
    text = model.generate(PROMPT, WAYS[way], {"onToken": lambda tok, i: alone.append((tok, i))})

    def on_token(tok, i):
        got.append((tok, i))
        scores.append(model.score(texts[i % len(texts)], 3))
    assert model.generate(PROMPT, WAYS[way], {"onToken": on_token}) == text
    assert got == alone and len(got) == 24
    for i, r in enumerate(scores):
        for name, x in want[(i + 1) % len(texts)].items():
            assert np.array_equal(r[name], x)
    assert model.generate(PROMPT, WAYS[way]) == text


@pytest.mark.parametrize("way", list(WAYS))
def test_scores_of_the_text_so_far(model, way):
    """A score of all that there is, at every token."""
    text, seen = model.generate(PROMPT, WAYS[way]), list(PROMPT)

    def on_token(tok, i):
        seen.append(tok)
        assert np.isfinite(model.score(seen)["logprobs"]).all()
    assert model.generate(PROMPT, WAYS[way], {"onToken": on_token}) == text == seen


@pytest.mark.parametrize("way", list(WAYS))
def test_steps_on_other_caches(model, way):
    vocab = model.config["vocabSize"]
    text = model.generate(PROMPT, WAYS[way])
    cache, own = model.createPagedCache(2, 80, 16, "f32"), model.createCache()

    def on_token(tok, i):
        if i % 3 == 0:
            model.scorePagedStep([[i % vocab], [5, 6]], cache, 4)
        elif i % 3 == 1:
            model.forwardPagedStep([[1, 2, 3], [tok]], cache)
        else:
            model.forwardPrefill(text[:i + 2], own)
            model.forwardDecode(7, i + 2, own)
    assert model.generate(PROMPT, WAYS[way], {"onToken": on_token}) == text
    cache.free()


def test_a_score_that_raises_ends_the_generation_only(model):
    """The next calls are as if there had been none."""
    text, score = model.generate(PROMPT, WAYS["greedy"]), model.score(PROMPT)

    def on_token(tok, i):
        model.score([tok] * (1 + (i < 5)))
    with pytest.raises(ValueError, match="score: a text of 1"):
        model.generate(PROMPT, WAYS["greedy"], {"onToken": on_token})
    assert model.generate(PROMPT, WAYS["greedy"]) == text
    assert np.array_equal(model.score(PROMPT)["logprobs"], score["logprobs"])
