"""cmf_qk_rope_dev and cmf_kv_copy_dev against their definitions in 64 bits.

Tolerance of the rotated heads: the mean of squares is summed in 64 bits and
its inverse root rounded to f32 (u = 2^-24 relative), two products with
roundings, then a c - b s with two products and a subtraction: at most 6 u of
|a| + |b|, |a|, |b| the normed elements; 16-bit rows add half a step of the
type relative to the value (f16: of its least normal below that)."""
import ctypes as C

import numpy as np
import pytest

from ops_util import rounded

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEP = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ops(gpu):
    from cmf_amd import ops
    return ops


def randn(r, *shape):
    return r.standard_normal(shape, dtype=np.float32)


def table(n):
    inv = 1e6 ** -(np.arange(64) / 64)
    ang = np.arange(n)[:, None] * inv
    return np.stack([np.cos(ang), np.sin(ang)], 2).astype(np.float32)


def turned(x, w, tab, pos, eps):
    """x [b][heads][128] f64 -> rotated, size |a| + |b| of each element."""
    y = x if w is None else x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * w
    a, b = y[..., :64], y[..., 64:]
    c, s = tab[pos][:, None, :, 0], tab[pos][:, None, :, 1]
    big = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, a * s + b * c], 2), np.concatenate([big, big], 2)


@pytest.mark.parametrize("b,nh,nkv,dtype,mode,norm", [
    (1, 16, 8, "float32", "cache", True), (1, 1, 1, "bfloat16", "cache", True), (5, 16, 8, "float32", "tree", True),
    (64, 32, 8, "float16", "tree", True), (37, 12, 4, "bfloat16", "cache", False), (700, 3, 1, "float32", "cache", True),
    (333, 8, 8, "float16", "cache", True), (2, 7, 3, "float32", "tree", False),
])
def test_qk_rope(ops, b, nh, nkv, dtype, mode, norm):
    T = ops.DevTensor
    r = np.random.default_rng(b + nh)
    pos0, eps = 41, 1e-6
    x = randn(r, b, nh + 2 * nkv + 1, 128)  # a padded row
    qn, kn = (1 + 0.2 * randn(r, 128) for _ in range(2))
    tab = table(pos0 + b + 3)
    depth = r.integers(0, b, b, dtype=np.int32) if mode == "tree" else None
    slots = pos0 + b + 9 if mode == "cache" else b + 2
    k, v = (T.of(np.full((nkv, slots, 128), 3.0, np.float32), dtype) for _ in range(2))
    q = T.of(np.full((b, nh + 1, 128), 4.0, np.float32))
    ops.qk_rope(T.of(x)[:, :nh + 2 * nkv], q[:, :nh], k, v, T.of(qn) if norm else None, T.of(kn) if norm else None, T.of(tab),
                pos0=pos0, depth=None if depth is None else T.of(depth), at_pos=mode == "cache", eps=eps)
    x, t = x.astype(np.float64), tab.astype(np.float64)
    pos = pos0 + (depth if depth is not None else np.arange(b))
    w = [n.astype(np.float64) if norm else None for n in (qn, kn)]
    wq, sq = turned(x[:, :nh], w[0], t, pos, eps)
    wk, sk = turned(x[:, nh:nh + nkv], w[1], t, pos, eps)
    wv = x[:, nh + nkv:nh + 2 * nkv]
    got = q.numpy()
    assert (np.abs(got[:, :nh] - wq) <= 6 * U * sq).all()
    assert (got[:, nh:] == 4.0).all()
    r0, st = pos0 if mode == "cache" else 0, STEP[dtype]
    for t, want, size in ((k, wk, sk), (v, wv, 0 * wv)):
        got = t.numpy().astype(np.float64)
        d = np.abs(got[:, r0:r0 + b] - want.transpose(1, 0, 2))
        tol = 6 * U * size + st * (np.abs(want) + 6 * U * size) + (2.0 ** -25 if dtype == "float16" else 0.0)
        assert (d <= tol.transpose(1, 0, 2)).all()
        rest = np.ones(slots, bool)
        rest[r0:r0 + b] = False
        assert (got[:, rest] == 3.0).all()


def test_qk_rope_one_side_and_rows_outside(ops, gpu):
    """Positions read on the device: rows past the table or the cache are left
    out, nothing else changes; queries or keys alone."""
    from cmf_amd import QkRopeArgs
    T = ops.DevTensor
    r = np.random.default_rng(3)
    b, nh, nkv, slots = 6, 4, 2, 20
    x, tab, nine = T.of(randn(r, b, 8, 128)), T.of(table(22)), lambda *s: T.of(np.full(s, 9.0, np.float32))
    full = [nine(b, nh, 128), nine(nkv, 40, 128), nine(nkv, 40, 128)]
    ops.qk_rope(x, *full, None, None, T.of(table(40)), pos0=17)
    q, k, v = nine(b, nh, 128), nine(nkv, slots, 128), nine(nkv, slots, 128)
    ops.qk_rope(x, q, k, v, None, None, tab, pos0=2, pos0_dev=T.of(np.array([15], np.int32)))  # positions 17 .. 22
    fq, fk, fv, gq, gk, gv = (t.numpy() for t in (*full, q, k, v))
    assert np.array_equal(gq[:5], fq[:5]) and (gq[5] == 9).all()
    assert np.array_equal(gk[:, 17:], fk[:, 17:20]) and np.array_equal(gv[:, 17:], fv[:, 17:20])
    assert (gk[:, :17] == 9).all() and (gv[:, :17] == 9).all()
    q2, k2 = nine(b, nh, 128), nine(nkv, slots, 128)
    common = dict(qkv=x.data_ptr(), rope=tab.data_ptr(), eps=1e-6, head_stride=slots * 128, row_stride=128, b=2, nh=nh, nkv=nkv,
                  ldq=1024, ldo=512, max_pos=22, pos0=17, slots=slots, at_pos=1)
    gpu.check(gpu.lib().cmf_qk_rope_dev(C.byref(QkRopeArgs(q_out=q2.data_ptr(), **common))))
    gpu.check(gpu.lib().cmf_qk_rope_dev(C.byref(QkRopeArgs(k=k2.data_ptr(), v=v.data_ptr(), **common))))
    hq, hk = q2.numpy(), k2.numpy()
    assert np.array_equal(hq[:2], gq[:2]) and (hq[2:] == 9).all()
    assert np.array_equal(hk[:, 17:19], gk[:, 17:19]) and (hk[:, 19:] == 9).all()


def ptrs(T, t):
    return T.of(np.array([t[i].data_ptr() for i in range(t.shape[0])], np.int64))


@pytest.mark.parametrize("bufs,nkv,n,dtype", [(1, 1, 1, "float32"), (56, 8, 5, "float32"), (3, 2, 64, "bfloat16"),
                                              (4, 3, 1001, "float16"), (2, 1, 777, "float32"), (7, 4, 16, "bfloat16")])
def test_kv_copy(ops, bufs, nkv, n, dtype):
    T = ops.DevTensor
    r = np.random.default_rng(n)
    src, dst = (rounded(randn(r, bufs, nkv, n + e, 128), dtype) for e in (13, 30))
    ds, dd = T.of(src, dtype), T.of(dst, dtype)
    idx = r.integers(0, n + 13, n, dtype=np.int32)  # the same row twice too
    dst[:, :, 11:11 + n] = src[:, :, idx]
    ops.kv_copy(ptrs(T, dd), ptrs(T, ds), dd[0], ds[0], n=n, pos0=11, idx=T.of(idx))
    assert np.array_equal(dd.numpy(), dst)
    # rows outside either side are left out; the count and the position from the device
    m = max(1, n // 2)
    idx[0], idx[-1] = -1, n + 13
    for i in range(m):
        if 0 <= idx[i] < n + 13 and 28 + i < n + 30:
            dst[:, :, 28 + i] = src[:, :, idx[i]]
    ops.kv_copy(ptrs(T, dd), ptrs(T, ds), dd[0], ds[0], n=n, pos0=-2, idx=T.of(idx), n_dev=T.of(np.array([m], np.int32)),
                pos0_dev=T.of(np.array([30], np.int32)))
    assert np.array_equal(dd.numpy(), dst)


def test_kv_copy_between_layouts_and_prefix(ops):
    """A prefix (no index) out of position-major buffers into head-major ones."""
    T = ops.DevTensor
    r = np.random.default_rng(4)
    src = randn(r, 2, 50, 4, 128)  # [buffer][row][head]
    ds, dd = T.of(src), T.of(np.zeros((2, 4, 60, 128), np.float32))
    ops.kv_copy(ptrs(T, dd), ptrs(T, ds), dd[0], ds[0].permute(1, 0, 2), n=50, pos0=10)
    got = dd.numpy()
    assert np.array_equal(got[:, :, 10:], src.transpose(0, 2, 1, 3)) and (got[:, :, :10] == 0).all()
