"""cmf_logprobs_dev against its definition in 64 bits.

Tolerance: a weight e^(x - m) is off by u |x - m| log2(e) and the exponential's
own error (2 u); sums of V of them in lanes and trees, as independent errors
lambda = 8 times sqrt(64) u; log Z moves by that relative error, the entropy by
it times the differences it averages; x - m rounds once."""
import math

import numpy as np
import pytest

from ops_util import Stream, rounded

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops(gpu):
    from cmf_amd import ops
    return ops


def definition(x, target, k):
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    z = e.sum(1)
    d = np.where(e > 0, x - m, 0.0)
    with np.errstate(invalid="ignore"):
        lp = x - m - np.log(z)[:, None]
    t = np.array([lp[r, t] if 0 <= t < x.shape[1] else np.nan for r, t in enumerate(target)])
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    return t, np.log(z) - (e * d).sum(1) / z, order, np.take_along_axis(lp, order, 1), 1 + np.sqrt((e * d * d).sum(1) / z)


def run(ops, x, target, k):
    T = ops.DevTensor
    rows = x.shape[0]
    lp, ent = (T.of(np.full(rows, 5.0, np.float32)) for _ in range(2))
    ids = T.of(np.full((rows, k), -7, np.int32)) if k else None
    top = T.of(np.full((rows, k), 5.0, np.float32)) if k else None
    ws = T.empty(max(16, ops.logprobs_workspace(x, k)), "uint8")
    ops.logprobs(x, T.of(np.asarray(target, np.int32)), lp, ent, ids, top, ws)
    return [None if t is None else t.numpy() for t in (lp, ent, ids, top)]


def close(got, want, tol):
    assert (np.isnan(got) == np.isnan(want)).all()
    fine = np.isfinite(want)
    other = ~fine & ~np.isnan(want)
    assert (got[other] == want[other]).all()
    d = np.abs(got[fine] - want[fine])
    assert (d <= np.broadcast_to(tol, want.shape)[fine]).all(), d.max()


def verify(ops, x, host, target, k):
    t, ent, ids, top, size = definition(host, target, k)
    lp_, ent_, ids_, top_ = run(ops, x, target, k)
    rel = (8 * math.sqrt(64) + 40) * U
    plain = lambda a: np.abs(np.where(np.isfinite(a), a, 0.0))  # noqa: E731
    close(lp_, t, rel * size + 2 * U * plain(t))
    close(ent_, ent, rel * size * 4 + 4 * U * plain(ent))
    if k:
        assert (ids_ == ids).all()
        close(top_, top, (rel * size)[:, None] + 2 * U * plain(top))


@pytest.mark.parametrize("rows,V,k,dtype", [
    (1, 1, 1, "float32"), (1, 2, 2, "bfloat16"), (2, 63, 63, "float32"), (3, 64, 64, "float16"), (5, 151936, 8, "float32"),
    (1, 151936, 64, "bfloat16"), (40, 4097, 20, "float32"), (7, 4095, 5, "float16"), (300, 1001, 1, "float32"),
    (2500, 257, 3, "bfloat16"), (17, 32000, 0, "float32"), (2, 200001, 64, "float32"), (600, 5000, 64, "float16"),
])
def test_logprobs(ops, rows, V, k, dtype):
    r = np.random.default_rng(V + rows)
    x = rounded(r.standard_normal((rows, V), dtype=np.float32) * 4, dtype)
    verify(ops, ops.DevTensor.of(x, dtype), x, r.integers(0, V, rows), k)


@pytest.mark.parametrize("off", [1, 3, 7])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_off_the_16_byte_boundary(ops, off, dtype):
    """Views into wider rows of an odd length; what lies around them is NaN."""
    r = np.random.default_rng(off)
    wide = np.full((9, 10001), np.nan, np.float32)
    x = rounded(r.standard_normal((9, 9000), dtype=np.float32) * 3, dtype)
    wide[:, off:off + 9000] = x
    verify(ops, ops.DevTensor.of(wide, dtype)[:, off:off + 9000], x, [0, 8999, 5, -1, 9000, 1, 2, 3, 2 ** 31 - 1], 12)


def test_orders_and_ties(ops):
    """Equal logits everywhere, ascending, descending, few distinct values, -0
    among zeros: the lowest id first."""
    V = 20000
    i = np.arange(V, dtype=np.float32)
    r = np.random.default_rng(2)
    x = np.stack([np.zeros(V), i * 1e-3, -i * 1e-3, r.integers(0, 3, V), np.where(i % 3 == 0, -0.0, 0.0),
                  np.full(V, -40.0)]).astype(np.float32)
    verify(ops, ops.DevTensor.of(x), x, [77] * 6, 64)


def test_masked_infinite_and_nan_logits(ops):
    V, inf = 9000, np.inf
    r = np.random.default_rng(5)
    x = r.standard_normal((7, V), dtype=np.float32) * 3
    x[0, 10:] = -inf                    # ten tokens left
    x[1] = -inf
    x[1, 4500] = -3.0                   # one token left
    x[2, :V // 2] = np.finfo(np.float32).min
    x[3, 8000:] = -inf
    t = [5, 4500, 8000, 8500, 1, 2, 3]
    verify(ops, ops.DevTensor.of(x[:4]), x[:4], t[:4], 12)
    x[4] = -inf                         # nothing left
    x[5, 100] = np.nan
    x[6, 200] = inf
    lp, ent, ids, top = run(ops, ops.DevTensor.of(x), t, 12)
    assert np.isnan(lp[4:]).all() and np.isnan(ent[4:]).all() and np.isnan(top[4:]).all()
    assert ids[4].tolist() == list(range(12))
    assert 100 not in ids[5] and ids[6, 0] == 200
    few = np.array([[np.nan, 1.0, np.nan, 2.0]], np.float32)
    assert run(ops, ops.DevTensor.of(few), t[:1], 4)[2].tolist() == [[3, 1, 0, 2]]


def test_parts_of_the_outputs(ops):
    T = ops.DevTensor
    r = np.random.default_rng(7)
    x = T.of(r.standard_normal((3, 50000), dtype=np.float32))
    t = T.of(np.array([1, 2, 3], np.int32))
    full = run(ops, x, [1, 2, 3], 6)
    ws = T.empty(1 << 20, "uint8")
    lp, ent, ids, top = T.empty(3), T.empty(3), T.empty((3, 6), "int32"), T.empty((3, 6))
    ops.logprobs(x, t, lp, None, None, None, ws)
    ops.logprobs(x, None, None, ent, None, None, ws)
    ops.logprobs(x, None, None, None, ids, None, ws)
    ops.logprobs(x, None, None, None, None, top, ws)
    for got, want in zip((lp, ent, ids, top), full):
        assert np.array_equal(got.numpy(), want)


def test_captured(ops):
    T = ops.DevTensor
    x, t = T.empty((4, 60000)), T.of(np.array([1, 2, 3, 4], np.int32))
    lp, ent, ids, top = T.empty(4), T.empty(4), T.empty((4, 9), "int32"), T.empty((4, 9))
    ws = T.empty(1 << 20, "uint8")
    s = Stream()
    graph = s.capture(lambda: ops.logprobs(x, t, lp, ent, ids, top, ws, stream=s.handle))
    for seed in range(3):
        x.buf.upload(np.random.default_rng(seed).standard_normal((4, 60000), dtype=np.float32) * 3)
        for o in (lp, ids):
            o.buf.upload(np.zeros(o.shape, o.dtype))
        s.replay(graph)
        for got, want in zip((lp, ent, ids, top), run(ops, x, [1, 2, 3, 4], 9)):
            assert np.array_equal(got.numpy(), want)
    s.drop(graph)
