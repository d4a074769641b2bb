"""forwardPagedStep with as many columns (row, head) as the attention kernel of
many rows takes: 256 rows of 32 heads."""
import numpy as np
import pytest

from smith_amd import device
from smith_amd.gguf_loader import loadGGUF
from llama_fixtures import write_tiny_llama
from test_gpu_paged_llama import BAR, off

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("gguf") / "wide.gguf")
    write_tiny_llama(p, dim=512, layers=2, heads=32, kv_heads=8, ffn=512, vocab=320, context=20000)
    return loadGGUF(p)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [8, 16])
def test_chunks_of_a_prompt(model, dtype, page):
    """A prompt of 600 tokens in chunks, the last beside another request's first
    rows, against the prompt alone; 256 rows of one request and of two."""
    rs = np.random.RandomState(6)
    prompt, other = rs.randint(0, 320, 600).tolist(), rs.randint(0, 320, 150).tolist()
    cache = model.createPagedCache(2, 800 // page + 2, page, dtype)
    alone = [model.forwardPrefill(t, model.createCache())["logits"] for t in (prompt, other)]
    steps = [[prompt[:256], []], [prompt[256:400], other[:112]], [prompt[400:599], other[112:]], [prompt[599:], []]]
    device.profile_kernels(True)
    try:
        for k, tokens in enumerate(steps):
            got = model.forwardPagedStep(tokens, cache)
            want = np.stack([alone[b][cache.lens[b] - 1] for b in got["requests"]])
            assert (off(got["logits"], want) <= BAR[dtype]).all(), (k, off(got["logits"], want))
            rows = device.profile_read("smith_paged_attention_rows_%s_" % dtype)[1]
            assert rows == (2 if k < 2 else 0)  # both layers of the steps of 256 rows
    finally:
        device.profile_kernels(False)
    cache.free()
