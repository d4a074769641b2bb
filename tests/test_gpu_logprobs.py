"""smith_logprobs against 64 bits: all types, any number of rows and tokens, rows
that are cut, ties, masks, what is not finite, graphs, refusals."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device
import paged_reference as R

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def last_error():
    return device.lib.smith_last_error(device.ctx()).decode()


def reference(x, tokens, top):
    """(logprobs, entropy, top ids, top logprobs, sum p |d|, sum p d^2, log l) in f64."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1, keepdims=True)
        d = x - m
        e = np.exp(d)
        l = e.sum(1, keepdims=True)
        p = e / l
        pd = np.where(e > 0, p * d, 0.0)
        lp = d - np.log(l)
        entropy = np.log(l)[:, 0] - pd.sum(1)
        ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
        return (np.take_along_axis(lp, np.maximum(tokens, 0), 1), entropy, ids, np.take_along_axis(lp, ids, 1),
                np.abs(pd).sum(1), np.where(e > 0, p * d * d, 0.0).sum(1), np.log(l)[:, 0], d)


def check(x, tokens, top, out):
    lp, entropy, ids, top_lp, A, B, log_l, d = reference(x, tokens, top)
    # A thread adds 1/256 of the row's terms or less and corrects its sums once a
    # chunk of 16; the joins add a few.  A term e^d is off by 2 EPS |d| (product and
    # constant) and 2 EPS, its product with d by EPS more.
    n = 1.5 * x.shape[1] / 256 + 80
    err_l = EPS * (n + 2 * A)
    err_log = err_l + 2 * EPS * (1 + np.abs(log_l))
    err_s = EPS * ((n + 2) * A + 2 * B)
    assert (np.abs(out["entropy"] - entropy) <= err_log + err_s + err_l * A + EPS * (np.abs(log_l) + 2 * A)).all()
    for got, want in ((out["logprobs"], lp), (out["topLogprobs"], top_lp)):
        with np.errstate(invalid="ignore"):
            bar = err_log[:, None] + 2 * EPS * (np.abs(want) + np.abs(log_l)[:, None])
            near = (np.abs(got - want) <= bar) | (got == want)
        assert near.all()
    assert np.array_equal(out["topIds"], ids)


def run(x, dtype, tokens, top):
    r = S.logProbs(R.upload(R.stored(x, dtype), dtype), R.upload(tokens.astype(np.int32)), top)
    device.sync()
    return {k: t.data.astype(np.float64) if t.dtype == "f32" else t.data for k, t in r.items()}


def case(seed, rows, vocab, given, dtype, size=2.5):
    rs = np.random.RandomState(seed)
    x = (rs.standard_normal((rows, vocab)) * size).astype(np.float32)
    return rs, R.value(R.stored(x, dtype), dtype), rs.randint(0, vocab, (rows, given))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,given,top", [
    (1, 1, 1, 1), (3, 2, 2, 2), (2, 63, 0, 5), (1, 64, 1, 64), (5, 65, 70, 64), (1, 1023, 1, 3), (2, 1024, 1, 64),
    (1, 1025, 3, 20), (3, 4095, 1, 1), (4, 4096, 1, 0), (3, 4097, 2, 17), (1, 32000, 1, 5), (7, 50003, 3, 20),
    (1, 131072, 1, 64), (1100, 5000, 1, 8), (513, 8193, 1, 64), (2050, 37, 1, 4), (1, 700001, 2, 13)])
def test_logprobs(dtype, rows, vocab, given, top):
    rs, x, tokens = case(rows + vocab, rows, vocab, given, dtype)
    check(x, tokens, top, run(x, dtype, tokens, top))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-3, 30.0, 3000.0])
def test_flat_and_steep_rows(dtype, size):
    rs, x, tokens = case(5, 6, 9001, 2, dtype, size)
    check(x, tokens, 33, run(x, dtype, tokens, 33))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("order", ["equal", "rising", "falling", "few", "zeros", "late", "one lane"])
@pytest.mark.parametrize("vocab,top", [(700, 64), (20011, 64), (20011, 7)])
def test_orders_and_ties(dtype, order, vocab, top):
    """Whatever order the values come in, and of equal ones the lower place."""
    rs, x, tokens = case(vocab, 2, vocab, 1, dtype)
    if order == "equal":
        x[:] = 1.5
    elif order == "rising":
        x = np.sort(x, 1)
    elif order == "falling":
        x = np.sort(x, 1)[:, ::-1].copy()
    elif order == "few":
        x = rs.randint(0, 5, x.shape).astype(np.float64)
    elif order == "zeros":
        x = np.where(rs.rand(*x.shape) < 0.5, 0.0, -0.0)
    elif order == "late":
        x[:, -top:] += 40
    else:
        x[:, (np.arange(vocab) // 8) % 64 == 5] += 40
    x = R.value(R.stored(x.astype(np.float32), dtype), dtype)
    check(x, tokens, top, run(x, dtype, tokens, top))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("share", [0.02, 0.5, 0.999])
def test_banned_tokens(dtype, share):
    rs, x, tokens = case(7, 5, 30011, 40, dtype)
    x[rs.rand(*x.shape) < share] = -np.inf
    x[:, 17] = 1.0
    x[1], x[1, 29000] = -np.inf, -3.0  # one token is left: its probability is 1
    tokens[1, 0] = 29000
    out = run(x, dtype, tokens, 20)
    check(x, tokens, 20, out)
    assert out["entropy"][1] == 0 and out["logprobs"][1, 0] == 0 and out["topIds"][1].tolist() == [29000] + list(range(19))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [33, 40000])
def test_rows_without_a_distribution(dtype, vocab):
    rs, x, tokens = case(9, 8, vocab, 2, dtype)
    x[1, vocab // 2] = np.nan
    x[3, vocab - 1] = np.inf
    x[4] = -np.inf
    x[6] = np.nan
    x[6, 5:8] = 1, 3, 2
    odd, fine = [1, 3, 4, 6], [0, 2, 5, 7]
    out = run(x, dtype, tokens, 6)
    check(x[fine], tokens[fine], 6, {k: v[fine] for k, v in out.items()})
    for k in ("logprobs", "entropy", "topLogprobs"):
        assert np.isnan(out[k][odd]).all(), k
    assert out["topIds"][6].tolist() == [6, 7, 5, -1, -1, -1]
    assert out["topIds"][3, 0] == vocab - 1 and out["topIds"][4].tolist() == list(range(6))
    assert out["topIds"][1].tolist() == [i for i in np.argsort(-np.where(np.isnan(x[1]), -np.inf, x[1]), kind="stable")[:6]]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (3, 5), (7, 1001)])
def test_strides_and_alignment(dtype, shift, extra):
    rows, vocab, top = 9, 10007, 11
    rs, x, tokens = case(11, rows, vocab, 2, dtype)
    ld = vocab + extra
    flat = np.full(shift + rows * ld, 99.0, np.float32)  # what lies between the rows would be likely
    at = shift + np.arange(rows)[:, None] * ld + np.arange(vocab)
    flat[at] = x
    t = R.upload(R.stored(flat, dtype), dtype)
    out = {"logprobs": S.create([rows, 2]), "entropy": S.create([rows]), "topIds": S.create([rows, top], "i32"),
           "topLogprobs": S.create([rows, top])}
    e = 4 if dtype == "f32" else 2
    device.check(device.lib.smith_logprobs(
        device.ops_ctx(), {"f32": 0, "f16": 1, "bf16": 2}[dtype], t.buffer + shift * e, ld, rows, vocab,
        R.upload(tokens.astype(np.int32)).buffer, 2, top, *[out[k].buffer for k in ("logprobs", "entropy", "topIds", "topLogprobs")]))
    device.sync()
    check(x, tokens, top, {k: v.data.astype(np.float64) if v.dtype == "f32" else v.data for k, v in out.items()})


def test_tokens_that_are_none_and_outside():
    rs, x, tokens = case(13, 4, 500, 3, "f32")
    tokens[1, 1] = -1
    out = run(x, "f32", tokens, 2)
    assert out["logprobs"][1, 1] == 0
    out["logprobs"][1, 1] = reference(x, tokens, 2)[0][1, 1]
    check(x, tokens, 2, out)
    for bad in (500, -2, 2 ** 31 - 1):
        tokens[2, 0] = bad
        r = S.logProbs(R.upload(x.astype(np.float32)), R.upload(tokens.astype(np.int32)), 2)
        assert device.lib.smith_sync(device.ctx()) == -1 and "row 2: a token outside the vocabulary" in last_error()
        device.sync()
        got = r["logprobs"].data
        assert np.isnan(got[2, 0]) and np.isfinite(got[:2]).all() and np.isfinite(got[2, 1:]).all()


def test_rows_beyond_32_bit_offsets():
    rows, vocab = 9000, 131072  # 4.7 GB
    t = S.create([rows, vocab], "f32")
    try:
        device.check(device.lib.smith_randn(device.ops_ctx(), t.buffer, rows * vocab, 3, 0, 2.0, 0.0))
        tokens = np.zeros((rows, 1), np.int32)
        tokens[:, 0] = np.arange(rows) * 7 % vocab
        r = S.logProbs(t, R.upload(tokens), 4)
        device.sync()
        pick = [0, 4000, rows - 1]
        x = np.stack([device.download(t.buffer + b * vocab * 4, vocab * 4, np.float32) for b in pick]).astype(np.float64)
        check(x, tokens[pick], 4, {k: v.data[pick].astype(np.float64) if v.dtype == "f32" else v.data[pick] for k, v in r.items()})
    finally:
        t.release()


def test_repeated_calls_are_the_same_bits():
    rs, x, tokens = case(15, 3, 131072, 2, "f32")
    first = run(x, "f32", tokens, 64)
    for _ in range(3):
        again = run(x, "f32", tokens, 64)
        for k in first:
            assert np.array_equal(first[k], again[k])


def test_two_graphs_on_one_scratch():
    ctx, steps = device.ops_ctx(), []
    for seed, (rows, vocab, top) in enumerate([(3, 60000, 20), (40, 9000, 5)]):
        rs, x, tokens = case(seed, rows, vocab, 1, "f32")
        t, k = R.upload(x.astype(np.float32)), R.upload(tokens.astype(np.int32))
        out = [S.create([rows, 1]), S.create([rows]), S.create([rows, top], "i32"), S.create([rows, top])]

        def call(t=t, k=k, out=out, rows=rows, vocab=vocab, top=top):
            device.check(device.lib.smith_logprobs(ctx, 0, t.buffer, vocab, rows, vocab, k.buffer, 1, top,
                                                   *[o.buffer for o in out]))
        call()
        steps.append([call, t, k, out, rows, vocab, top, None])
    device.sync()
    try:
        for st in steps:
            device.check(device.lib.smith_graph_begin(ctx), "begin")
            st[0]()
            st[-1] = device.lib.smith_graph_end(ctx)
            assert st[-1], last_error()
        for turn in range(4):
            want = []
            for st in steps:
                rs, x, tokens = case(100 + turn, st[4], st[5], 1, "f32")
                st[1].set_data(x), st[2].set_data(tokens)
                want.append((x, tokens))
            for st in steps:
                device.check(device.lib.smith_graph_launch(ctx, st[-1]))
            for st, (x, tokens) in zip(steps, want):
                got = [o.data for o in st[3]]
                check(x, tokens, st[6], {"logprobs": got[0].astype(np.float64), "entropy": got[1].astype(np.float64),
                                         "topIds": got[2], "topLogprobs": got[3].astype(np.float64)})
            steps[0][0]()  # eager, between
            device.sync()
    finally:
        for st in steps:
            if st[-1]:
                device.lib.smith_graph_destroy(st[-1])


_arena = []


@pytest.mark.parametrize("over,message", [
    ({"type": 3}, "unknown type of logits 3"), ({"vocab": 0}, "a vocabulary of 0"), ({"vocab": 1 << 31, "ld": 1 << 31}, "a vocabulary of"),
    ({"ld": 99}, "row stride 99"), ({"rows": 1 << 31}, "rows"), ({"given": 1 << 31}, "tokens each"), ({"top": 65}, "65 top"),
    ({"vocab": 3, "top": 4}, "4 top"), ({"x": None}, "null buffer"), ({"tokens": None}, "null buffer"), ({"lp": None}, "null buffer"),
    ({"ids": None}, "null buffer"), ({"tlp": None}, "null buffer"), ({"x": 4098}, "not aligned"), ({"lp": 4096}, "overlaps an input"),
    ({"ent": 4096 + 1196}, "overlaps an input"), ({"ids": 65536}, "overlaps an input"), ({"tlp": 1 << 17}, "two outputs overlap"),
    ({"ent": (1 << 17) + 20}, "two outputs overlap")])
def test_refusals(over, message):
    a = dict(type=0, x=4096, ld=100, rows=3, vocab=100, tokens=65536, given=2, top=5, lp=1 << 17, ent=(1 << 17) + 64,
             ids=(1 << 17) + 128, tlp=(1 << 17) + 256)
    a.update(over)
    if not _arena:
        _arena.append(S.zeros([1 << 18], "i32"))
    for k in ("x", "tokens", "lp", "ent", "ids", "tlp"):
        a[k] = a[k] if a[k] is None else _arena[0].buffer + a[k]
    assert device.lib.smith_logprobs(device.ops_ctx(), *a.values()) == -1
    assert "smith_logprobs: " in last_error() and message in last_error()


def test_calls_of_nothing():
    ctx = device.ops_ctx()
    assert device.lib.smith_logprobs(ctx, 0, None, 5, 0, 5, None, 0, 0, None, None, None, None) == 0
    x = S.ones([2, 5])
    assert device.lib.smith_logprobs(ctx, 0, x.buffer, 5, 2, 5, None, 0, 0, None, None, None, None) == 0
    device.sync()


def test_wrapper_refusals():
    x = S.ones([2, 5])
    for args, message in (((S.ones([5]),), "logits are"), ((x, S.zeros([3], "i32")), "tokens are"), ((x, S.zeros([2])), "tokens are"),
                          ((x, None, 6), "6 top"), ((x, None, -1), "-1 top")):
        with pytest.raises(ValueError, match="logProbs: .*" + message):
            S.logProbs(*args)
