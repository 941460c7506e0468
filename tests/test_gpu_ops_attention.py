"""cmf_attention_dev against its definition in 64 bits: trees and chains over a
cache, windows with sinks, the storage types, head layouts, odd sizes and
strides, rows that see nothing, garbage where nothing looks.

Tolerance: a score is a dot of 128 products in f32, off by about lambda
sqrt(128) u |q||k| scale (u = 2^-24, rounding errors as independent, lambda =
8), which moves every weight by that relative amount (numerator and
denominator: twice); the sums over n keys add lambda sqrt(n) u, and a weight is
2^(s log2 e) of a score of size s, which rounding moves by u s.  An output is at
most max |v| of what the row sees."""
import math

import numpy as np
import pytest

from ops_util import Stream, rounded

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HD = 128


def randn(r, *shape):
    return r.standard_normal(shape, dtype=np.float32)


def tensors(r, b, ctx, nh, nkv, dtype, extra=0, std=1.5):
    q = randn(r, b, nh, HD) * np.float32(std)
    k, v = (rounded(randn(r, nkv, ctx + extra, HD), dtype) for _ in range(2))
    return q, k, v


def visible(b, ctx, window, sinks, mask=None, depth=None):
    """[b][ctx + b]: cached positions, then the new rows."""
    see = np.zeros((b, ctx + b), bool)
    for i in range(b):
        P = ctx + (int(depth[i]) if depth is not None else i)
        x = np.arange(ctx + b)
        near = (x > P - window) | (x < sinks) if window else np.ones(ctx + b, bool)
        see[i] = near & (x <= ctx + i)
        if mask is not None:
            see[i, ctx:] = [(int(mask[i]) >> j) & 1 for j in range(b)]
    return see


def reference(q, k, v, see, scale=HD ** -0.5):
    """q [b][nh][128], k / v [nkv][keys][128] -> out and tolerance in f64."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    b, nh, _ = q.shape
    nkv = k.shape[0]
    hpk = nh // nkv
    out, tol = np.zeros((b, nh, HD)), np.zeros((b, nh, 1))
    for i in range(b):
        x = np.flatnonzero(see[i])
        if not len(x):
            continue
        for g in range(nkv):
            kk, vv = k[g, x], v[g, x]
            qq = q[i, g * hpk:(g + 1) * hpk]
            s = qq @ kk.T * scale
            p = np.exp(s - s.max(1, keepdims=True))
            out[i, g * hpk:(g + 1) * hpk] = p @ vv / p.sum(1, keepdims=True)
            size = np.linalg.norm(qq, axis=1) * np.linalg.norm(kk, axis=1).max() * abs(scale)
            tol[i, g * hpk:(g + 1) * hpk, 0] = np.abs(vv).max() * (
                2 * 8 * math.sqrt(128) * U * size + 8 * math.sqrt(len(x)) * U + 4 * U * np.abs(s).max(1) + 8 * U)
    return out, tol


def check(got, want, tol):
    assert np.isfinite(got).all()
    d = np.abs(got.astype(np.float64) - want)
    assert (d <= tol).all(), (d / np.maximum(tol, 1e-300)).max()


def random_tree(b, seed):
    r = np.random.RandomState(seed)
    return [-1] + [int(r.randint(max(0, i - 6), i)) for i in range(1, b)]


@pytest.fixture(scope="module")
def ops(gpu):
    from cmf_amd import ops
    return ops


@pytest.fixture(scope="module")
def ws(ops):
    return ops.DevTensor.empty(64 << 20, "uint8")


def filled(ops, shape, x=7.0):
    return ops.DevTensor.of(np.full(shape, x, np.float32))


def run_tree(ops, ws, q, k, v, kn, vn, dtype, ctx, mask, depth, window=0, sinks=0):
    T = ops.DevTensor
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx, k_new=T.of(kn, dtype), v_new=T.of(vn, dtype),
                  mask=T.of(mask), depth=T.of(depth), window=window, sinks=sinks)
    return out.numpy()


@pytest.mark.parametrize("b,ctx,nh,nkv,dtype", [
    (1, 0, 2, 2, "float32"), (1, 1, 16, 8, "float32"), (2, 0, 4, 1, "bfloat16"), (5, 63, 16, 8, "float32"),
    (9, 64, 12, 4, "float16"), (9, 2048, 16, 8, "float32"), (17, 65, 8, 8, "bfloat16"), (29, 1201, 16, 8, "float32"),
    (33, 500, 32, 2, "float16"), (64, 3001, 32, 8, "bfloat16"), (64, 0, 8, 1, "float32"), (64, 129, 3, 1, "float32"),
    (64, 4099, 64, 1, "float32"), (7, 20011, 5, 5, "float16"), (64, 5001, 64, 2, "bfloat16"), (64, 5001, 64, 1, "float16"),
    (29, 12001, 16, 8, "float32"), (3, 300, 600, 600, "float32"), (1, 4001, 300, 300, "bfloat16"),
])
def test_tree(ops, ws, b, ctx, nh, nkv, dtype):
    r = np.random.default_rng(b * 1000 + ctx)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype)
    _, kn, vn = tensors(r, b, b, nh, nkv, dtype)
    mask, depth = ops.tree_masks(random_tree(b, ctx))
    out = run_tree(ops, ws, q, k, v, kn, vn, dtype, ctx, mask, depth)
    see = visible(b, ctx, 0, 0, mask, depth)
    check(out, *reference(q, np.concatenate([k, kn], 1), np.concatenate([v, vn], 1), see))


@pytest.mark.parametrize("b,ctx,window,sinks,nh,nkv,dtype", [
    (1, 0, 1, 0, 16, 8, "float32"), (1, 5000, 1, 0, 16, 8, "float32"), (1, 5000, 1, 1, 4, 4, "float32"),
    (1, 12000, 1024, 4, 16, 8, "float32"), (3, 100, 64, 37, 8, 1, "bfloat16"), (16, 100, 200, 4, 16, 8, "float32"),
    (16, 1000, 17, 1000, 16, 4, "float16"), (200, 0, 0, 0, 16, 8, "float32"), (130, 70, 33, 5, 16, 8, "float32"),
    (257, 1000, 128, 4, 12, 4, "bfloat16"), (512, 31, 100, 128, 16, 8, "float32"), (300, 200, 16, 0, 2, 1, "float16"),
    (65, 0, 1, 0, 4, 2, "float32"), (700, 3, 64, 1, 8, 8, "float32"), (90, 4000, 0, 0, 12, 4, "float32"),
    (900, 2500, 0, 0, 16, 8, "float32"), (1000, 3001, 1500, 70, 12, 4, "bfloat16"), (900, 1000, 1700, 130, 16, 4, "float16"),
])
def test_window(ops, ws, b, ctx, window, sinks, nh, nkv, dtype):
    T = ops.DevTensor
    r = np.random.default_rng(b * 77 + ctx + window)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype, extra=b)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx, window=window, sinks=sinks)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, window, sinks)))


@pytest.mark.parametrize("b,ctx,window,sinks", [(40, 50, 6, 3), (64, 300, 64, 0), (9, 4, 3, 7), (24, 2000, 1, 0),
                                                (64, 2000, 1500, 40)])
def test_tree_under_a_window(ops, ws, b, ctx, window, sinks):
    r = np.random.default_rng(b)
    q, k, v = tensors(r, b, ctx, 16, 8, "float32")
    _, kn, vn = tensors(r, b, b, 16, 8, "float32")
    mask, depth = ops.tree_masks(random_tree(b, 3), pos0=ctx, window=window, sinks=sinks)
    out = run_tree(ops, ws, q, k, v, kn, vn, "float32", ctx, mask, depth, window, sinks)
    see = visible(b, ctx, window, sinks, mask, depth)
    check(out, *reference(q, np.concatenate([k, kn], 1), np.concatenate([v, vn], 1), see))


@pytest.mark.parametrize("b,nh,nkv", [(6, 16, 8), (60, 16, 4)])
def test_rows_that_see_nothing(ops, ws, b, nh, nkv):
    r = np.random.default_rng(1)
    q, kn, vn = tensors(r, b, b, nh, nkv, "float32")
    k = np.zeros((nkv, 4, HD), np.float32)
    mask = np.arange(b, dtype=np.uint64) % 3  # rows 0, 3, ..: nothing
    out = run_tree(ops, ws, q, k, k, kn, vn, "float32", 0, mask, np.zeros(b, np.int32))
    see = np.array([[(int(m) >> j) & 1 == 1 for j in range(b)] for m in mask])
    check(out, *reference(q, kn, vn, see))
    assert (out[::3] == 0).all()


def test_rows_past_every_key_of_their_window(ops, ws):
    """Rows of a large tree so deep that nothing of a long cache is near, with
    an empty mask: zeros; the others see the cache."""
    b, ctx, window, nh = 64, 1000, 900, 64
    r = np.random.default_rng(15)
    q, k, v = tensors(r, b, ctx, nh, 1, "float32")
    _, kn, vn = tensors(r, b, b, nh, 1, "float32")
    mask = np.array([0 if i % 5 == 2 else 1 << i for i in range(b)], np.uint64)
    depth = np.array([5000 if i % 5 == 2 else i for i in range(b)], np.int32)
    out = run_tree(ops, ws, q, k, v, kn, vn, "float32", ctx, mask, depth, window)
    see = visible(b, ctx, window, 0, mask, depth)
    check(out, *reference(q, np.concatenate([k, kn], 1), np.concatenate([v, vn], 1), see))
    assert (out[2::5] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("b,nh,nkv,dtype,ctx,window", [
    (5, 16, 8, "float32", 200, 90), (9, 4, 2, "float16", 200, 90), (64, 16, 4, "float32", 200, 90),
    (64, 16, 4, "bfloat16", 200, 90), (64, 64, 1, "float32", 1400, 1200), (64, 64, 1, "bfloat16", 3400, 3100),
    (64, 64, 1, "float16", 3400, 3100)])
def test_garbage_where_a_row_does_not_look(ops, ws, b, nh, nkv, dtype, ctx, window, bad):
    """A tree row that other rows do not see, cache rows behind the window and
    past the end hold NaN or infinities: only the row that sees them feels it."""
    sinks = 3
    r = np.random.default_rng(5)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype, extra=60)
    _, kn, vn = tensors(r, b, b, nh, nkv, dtype)
    mask, depth = ops.tree_masks([-1] + [(i - 1) // 2 for i in range(1, b)], pos0=ctx, window=window, sinks=sinks)
    hurt = b - 1  # a leaf: seen by itself alone
    see = visible(b, ctx, window, sinks, mask, depth)
    want, tol = reference(q, np.concatenate([k[:, :ctx], kn], 1), np.concatenate([v[:, :ctx], vn], 1), see)
    for t in (k, v):
        t[:, ctx:] = bad                      # past the end
        t[:, sinks:ctx - window + 1] = bad    # behind every row's window
    for t in (kn, vn):
        t[:, hurt] = bad
    out = run_tree(ops, ws, q, k, v, kn, vn, dtype, ctx, mask, depth, window, sinks)
    rows = [i for i in range(b) if i != hurt]
    check(out[rows], want[rows], tol[rows])
    if bad != -float("inf"):  # (a key of -inf may have a score of -inf: a weight of 0)
        assert not np.isfinite(out[hurt]).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("b,window", [(160, 20), (1600, 1000)])
def test_garbage_seen_by_some_rows_of_a_chunk(ops, ws, b, window, bad, what):
    """Row 40 of a chunk holds garbage: the rows from it see it through their
    window, the others do not."""
    T = ops.DevTensor
    r = np.random.default_rng(6)
    ctx, last = 10, 40 + window
    q, k, v = tensors(r, b, ctx, 16, 8, "float32", extra=b)
    want, tol = reference(q, k, v, visible(b, ctx, window, 0))
    (k if what == "k" else v)[:, ctx + 40] = bad
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k), T.of(v), out, ws, pos0=ctx, window=window)
    out = out.numpy()
    rows = [i for i in range(b) if not 40 <= i < last]
    check(out[rows], want[rows], tol[rows])
    assert not np.isfinite(out[40:last]).any()


@pytest.mark.parametrize("big", [1e4, 1e10, 1e30])
@pytest.mark.parametrize("b,nh,nkv,ctx,window", [(5, 16, 4, 300, 280), (64, 16, 4, 300, 280), (64, 64, 1, 1300, 1280)])
def test_values_of_another_size_seen_by_some_rows(ops, ws, b, nh, nkv, ctx, window, big):
    """A leaf of a tree, and a cached position that only the first rows see
    through their window, hold values `big` times the others': the rows that do
    not see them keep their accuracy."""
    r = np.random.default_rng(13)
    q, k, v = tensors(r, b, ctx, nh, nkv, "float32")
    _, kn, vn = tensors(r, b, b, nh, nkv, "float32")
    mask, depth = ops.tree_masks([-1] + [max(0, i - 2) for i in range(1, b)], pos0=ctx, window=window)
    v[:, ctx - window + 1] *= np.float32(big)  # seen at depth 0 alone
    vn[:, b - 1] *= np.float32(big)
    see = visible(b, ctx, window, 0, mask, depth)
    want, tol = reference(q, np.concatenate([k, kn], 1), np.concatenate([v, vn], 1), see)
    out = run_tree(ops, ws, q, k, v, kn, vn, "float32", ctx, mask, depth, window)
    check(out, want, tol)


@pytest.mark.parametrize("size", [1e-18, 1e18])
@pytest.mark.parametrize("b,ctx", [(4, 300), (64, 300), (1000, 1500)])
def test_far_ranges(ops, ws, b, ctx, size):
    """Keys and values of 1e18 (1e-18) against queries of 1e-18 (1e18)."""
    T = ops.DevTensor
    r = np.random.default_rng(8)
    q, k, v = tensors(r, b, ctx, 8, 2, "float32", extra=b)
    q, k, v = q / np.float32(size), k * np.float32(size), v * np.float32(size)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k), T.of(v), out, ws, pos0=ctx)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, 0, 0)))


@pytest.mark.parametrize("b,ctx", [(1, 777), (40, 777), (150, 333), (1500, 333)])
@pytest.mark.parametrize("stream", [None, 0])
def test_strides_scale_and_a_position_on_the_device(ops, ws, b, ctx, stream):
    """A cache whose positions are interleaved with other data, padded query and
    output rows, a scale of its own, the position read on the device (larger
    bound), on the library's stream and the null stream: what lies between the
    rows stays."""
    T = ops.DevTensor
    r = np.random.default_rng(9)
    nh, nkv, slots = 12, 4, ctx + b + 100
    kc, vc = (randn(r, slots, 2, nkv, HD) for _ in range(2))  # [slot][which][head]
    qc = randn(r, b, nh + 3, HD)
    dk, dv = (T.of(t)[:, 0].permute(1, 0, 2) for t in (kc, vc))
    out = filled(ops, (b, nh + 2, HD), 5.0)
    ops.attention(T.of(qc)[:, 1:nh + 1], dk, dv, out[:, :nh], ws, pos0=7, pos0_dev=T.of(np.array([ctx - 7], np.int32)),
                  len_bound=ctx + 90, window=150, sinks=2, scale=0.05, stream=stream)
    if stream == 0:
        Stream().hip.hipStreamSynchronize(None)
    got = out.numpy()
    k, v = (t[:ctx + b, 0].transpose(1, 0, 2) for t in (kc, vc))
    check(got[:, :nh], *reference(qc[:, 1:nh + 1], k, v, visible(b, ctx, 150, 2), 0.05))
    assert (got[:, nh:] == 5.0).all()


def test_offsets_past_32_bits(ops, ws):
    """The last positions of a cache whose last head starts 8.6 GB in."""
    import ctypes as C

    import cmf_amd
    T = ops.DevTensor
    ctx, b, nkv, n = 2_100_000, 3, 9, 103
    r = np.random.default_rng(10)
    lo = ctx + b - n
    k, v = (T.empty((nkv, ctx + b, HD)) for _ in range(2))
    assert k.stride()[0] * (nkv - 1) * 4 > 1 << 33
    tail = [randn(r, nkv, n, HD) for _ in range(2)]
    for t, x in ((k, tail[0]), (v, tail[1])):
        for g in range(nkv):
            row = np.ascontiguousarray(x[g])
            cmf_amd.check(cmf_amd.lib().cmf_h2d(t[g, lo:].data_ptr(), row.ctypes.data_as(C.c_void_p), row.nbytes))
    q = randn(r, b, 2 * nkv, HD)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), k, v, out, ws, pos0=ctx, window=100)
    see = np.array([[lo + j > ctx + i - 100 and lo + j <= ctx + i for j in range(n)] for i in range(b)])
    check(out.numpy(), *reference(q, tail[0], tail[1], see))


@pytest.mark.parametrize("b,tree", [(1, False), (12, True), (64, True), (200, False), (700, False)])
def test_captured_calls(ops, b, tree):
    """Two captured calls with a scratch each, replayed with other positions and
    eager calls between: every replay equals the eager call, bit for bit."""
    T = ops.DevTensor
    r = np.random.default_rng(11)
    q, k, v = (T.of(t) for t in tensors(r, b, 1200 + b, 16, 8, "float32"))
    _, kn, vn = (T.of(t) for t in tensors(r, b, b, 16, 8, "float32"))
    at = T.of(np.array([100], np.int32))
    kw = dict(pos0_dev=at, len_bound=1200)
    if tree:
        mask, depth = ops.tree_masks(random_tree(b, 2))
        kw.update(mask=T.of(mask), depth=T.of(depth), k_new=kn, v_new=vn)
    s = Stream()
    scr = [T.empty(64 << 20, "uint8") for _ in range(3)]
    outs = [filled(ops, q.shape) for _ in range(3)]
    kinds = ({}, dict(window=64, sinks=4))

    def both():
        for i, w in enumerate(kinds):
            ops.attention(q, k, v, outs[i], scr[i], stream=s.handle, **kw, **w)
    graph = s.capture(both)
    for p in (100, 0, 1200, 513):
        at.buf.upload(np.array([p], np.int32))
        for o in outs:
            o.buf.upload(np.full(q.shape, 3, np.float32))
        s.replay(graph)
        for i, w in enumerate(kinds):
            ops.attention(q, k, v, outs[2], scr[2], **kw, **w)
            assert np.array_equal(outs[2].numpy(), outs[i].numpy()), (p, i)
    s.drop(graph)


def test_a_scratch_too_small_is_refused(ops):
    import cmf_amd
    T = ops.DevTensor
    r = np.random.default_rng(12)
    q, k, v = (T.of(t) for t in tensors(r, 1, 5001, 16, 8, "float32"))
    out = filled(ops, q.shape, 2.0)
    need = ops.attention_workspace(q, k, v, pos0=5000)
    assert need > 0
    with pytest.raises(cmf_amd.CmfError, match="workspace"):
        ops.attention(q, k, v, out, None, pos0=5000)
    with pytest.raises(cmf_amd.CmfError, match="workspace"):
        ops.attention(q, k, v, out, T.empty(need - 1, "uint8"), pos0=5000)
    assert (out.numpy() == 2.0).all()
    ops.attention(q, k, v, out, T.empty(need, "uint8"), pos0=5000)
    assert not (out.numpy() == 2.0).any()


@pytest.mark.parametrize("b,ctx,window,sinks,nh,nkv,dtype", [
    (1030, 500, 0, 0, 32, 16, "float32"), (2060, 40, 600, 4, 16, 16, "float16"), (2060, 900, 0, 0, 16, 16, "bfloat16")])
def test_blocks_that_do_not_fill_the_card(ops, ws, b, ctx, window, sinks, nh, nkv, dtype):
    """272 blocks of 128 queries: as tiles, 256 in one piece and the rest split over
    their keys."""
    T = ops.DevTensor
    r = np.random.default_rng(b + ctx)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype, extra=b)
    out = filled(ops, q.shape)
    dq, dk, dv = T.of(q), T.of(k, dtype), T.of(v, dtype)
    ops.attention(dq, dk, dv, out, ws, pos0=ctx, window=window, sinks=sinks)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, window, sinks)))


@pytest.mark.parametrize("b", [1, 9, 80, 900])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_of_1e36(ops, ws, b, dtype):
    """weights are summed without leaving f32's range"""
    T = ops.DevTensor
    r = np.random.default_rng(b)
    q, k, v = tensors(r, b, 700, 4, 2, dtype, extra=b, std=4.0)
    v = rounded(v * np.float32(1e36), dtype)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=700)
    check(out.numpy(), *reference(q, k, v, visible(b, 700, 0, 0)))


@pytest.mark.parametrize("b,ctx", [(1, 100), (5, 3000), (1000, 1500)])
def test_output_over_the_queries(ops, ws, b, ctx):
    T = ops.DevTensor
    r = np.random.default_rng(b)
    q, k, v = (T.of(t) for t in tensors(r, b, ctx, 16, 8, "float32", extra=b))
    out = filled(ops, q.shape)
    ops.attention(q, k, v, out, ws, pos0=ctx)
    ops.attention(q, k, v, q, ws, pos0=ctx)
    assert np.array_equal(q.numpy(), out.numpy())
