"""Scores of tokens: what a model's logits say about given tokens and which ones
it would rather have, without the logits leaving the device.

The reference samples on the host from downloaded logits (generate.js:11-70) and
has no scores; logProbs is one call into libsmith.so (smith_logprobs,
include/smith.h).
"""
from . import device
from . import tensor as T

LOGIT_TYPES = {"f32": 0, "f16": 1, "bf16": 2}
MAX_TOP = 64


def logProbs(logits, tokens=None, top=0):
    """Of logits [rows, vocab] (f32, f16 or bf16) {logprobs [rows, given], entropy
    [rows], topIds, topLogprobs [rows, top]} as new Tensors: the log probabilities
    of tokens [rows] or [rows, given] i32 (-1: none, 0), the entropy, and the top
    <= 64 alternatives, the likeliest first (smith_logprobs)."""
    if logits.dtype not in LOGIT_TYPES or len(logits.shape) != 2:
        raise ValueError("logProbs: logits are [rows, vocab] of f32, f16 or bf16, got %s %s" % (logits.dtype, logits.shape))
    rows, vocab = logits.shape
    given = 0
    if tokens is not None:
        if tokens.dtype != "i32" or len(tokens.shape) not in (1, 2) or tokens.shape[0] != rows:
            raise ValueError("logProbs: tokens are i32 [%d] or [%d, given], got %s %s" % (rows, rows, tokens.dtype, tokens.shape))
        given = tokens.shape[1] if len(tokens.shape) == 2 else 1
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError("logProbs: %d top alternatives of a vocabulary of %d (up to %d)" % (top, vocab, MAX_TOP))
    out = {"logprobs": T.create([rows, given]), "entropy": T.create([rows]), "topIds": T.create([rows, top], "i32"),
           "topLogprobs": T.create([rows, top])}
    device.check(device.lib.smith_logprobs(
        device.ops_ctx(), LOGIT_TYPES[logits.dtype], logits.buffer, vocab, rows, vocab,
        tokens.buffer if given else None, given, top, out["logprobs"].buffer, out["entropy"].buffer,
        out["topIds"].buffer, out["topLogprobs"].buffer), "logProbs")
    return out
