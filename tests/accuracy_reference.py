"""How far attention in f32 accuracy is from 64 bits, as a norm over many outputs.

Of q of standard deviation 2 and keys of 1 a score S has deviation 2 and the largest
of some hundred keys is about 8.  Of an output sum p v / sum p the error is that of
its weights, relative: ||error|| / ||out|| is the root mean square d of what a weight
is off by, since both are sums over the same keys with the same weights and values of
either sign.  In steps of u = 2^-24 (a value in [1, 2) is off by up to u, 0.58 u in the
mean square):
  q in parts, to 2^-22 of the row's largest element (6): 6 * 4u * 0.58 / 2, through D
    elements, keys of 1 and the scale 1 / sqrt(D)              7 u
  the score, D / 4 sums of up to 4 in magnitude (f32 products) 0.58 * 1.2 * sqrt(D / 4) = 4 u
  S log2 e - m, of up to 16, and its product: 0.58 * 8 * ln 2  3.2 u
  the exponential, the weight's parts                          2 u
  the sums of n <= 1500 keys, a quarter of them a wave's, 16 at a time: 0.58 * sqrt(n / 16) 6 u
together less than 11 u = 7e-7, and the bar is three times that.  Of q of deviation 1/4
the first three are an eighth, together less than 7 u = 4e-7, and the bar is twice that.
A part of q that is lost shows above the first bar, and a part of the weights above the
second (test_accuracy_host.py)."""
import numpy as np

BARS = {2.0: 2e-6, 0.25: 8e-7}  # by q's deviation


def check_norm(got, want, keys, q_std):
    """Of rows of the sizes above, those that see 30 keys and more (one that sees few has a
    larger norm and hides the others): the root mean square of what they are off by."""
    rows = np.asarray(keys) >= 30
    want = want.reshape(len(rows), -1)
    off = np.linalg.norm(got.astype(np.float64).reshape(want.shape) - want, axis=1)[rows] / np.linalg.norm(want, axis=1)[rows]
    off = np.sqrt((off ** 2).mean())
    assert off <= BARS[q_std], off


def parts(x, dtype, terms):
    """x (f64) as the sum of so many numbers of dtype, each what is left of it, to nearest."""
    out = np.zeros_like(x)
    for _ in range(terms):
        rest = x - out
        if dtype == "f16":
            out = out + rest.astype(np.float16).astype(np.float64)
        else:  # bf16: 8 bits of the significand
            m, e = np.frexp(rest)
            out = out + np.ldexp(np.rint(m * 256) / 256, e)
    return out


def attention(q, k, v, dtype=None, q_terms=0, p_terms=0):
    """Of rows q [rows, D] over k, v [keys, D] in 64 bits, q (against its row's largest
    element) and the weights held in so many parts of dtype."""
    if q_terms:
        top = np.ldexp(1.0, np.frexp(np.abs(q).max(1, keepdims=True))[1])
        q = parts(q / top, dtype, q_terms) * top
    s = q @ k.T / np.sqrt(q.shape[1])
    p = np.exp(s - s.max(1, keepdims=True))
    out = (parts(p, dtype, p_terms) if p_terms else p) @ v
    return out / p.sum(1, keepdims=True)
