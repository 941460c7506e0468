"""cmf_attention_dev where the sizes of queries, keys, values and scores differ
within a call: what a row does not see may be of any size, and neither kernel
may lose what it does see.  Sizes take the kernel of few queries and the one of
tiles, whole and split over the keys.

Tolerances are those of test_gpu_ops_attention.py: by the largest key and value
that a row sees, so that they stay tight for the rows that see ordinary ones."""
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT
from ops_util import rounded
from test_gpu_ops_attention import HD, U, check, filled, ops, reference, run_tree, tensors, visible, ws  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- scores ---------------------------------------------------------------
@pytest.mark.parametrize("power", [3, 8, 12, 20, 30])
@pytest.mark.parametrize("b,ctx,nh,nkv,dtype", [
    (5, 300, 16, 8, "float32"), (9, 3000, 16, 8, "float16"), (3, 500, 4, 2, "bfloat16"), (64, 300, 16, 4, "float32"),
    (64, 3000, 64, 1, "bfloat16"), (1000, 1500, 16, 8, "float32"), (1000, 1500, 16, 8, "float16")])
def test_large_scores(ops, ws, b, ctx, nh, nkv, dtype, power):
    """Queries and keys of 1 and -1 in their first 6 dims times 2^power: scores
    are exact in f32, distinct ones lie at least 2^(2 power - 2) apart.  For the
    larger powers the weights are 1 for the keys that share a row's largest
    score and 0 for all others: the output is those values' mean, rounded like
    any sum (2^-24 of the largest value for each of its sqrt(n) independent
    roundings, 8 fold, and a few for the operands in parts)."""
    T = ops.DevTensor
    r = np.random.default_rng(b + ctx + power)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype, extra=b)
    most = 12 if dtype == "float16" else 60
    for t, p in ((q, 2 * power - min(power, most)), (k, min(power, most))):
        t[...] = np.where(t < 0, -1, 1)
        t[..., 6:] = 0
        t *= np.float32(2.0 ** p)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx, scale=0.125)
    want, tol = reference(q, k, v, visible(b, ctx, 0, 0), 0.125)
    if power > 3:  # (one step between scores is 2^14 at least: e^-2^14 is 0)
        tol = np.abs(v).max() * U * (8 * np.sqrt(ctx + b) + 16) + 0 * tol
    check(out.numpy(), want, tol)


@pytest.mark.parametrize("power", [6, 12, 14, 15, 16, 20, 30])
@pytest.mark.parametrize("sizes", [(0.01,), (1e-9,), (300.0,), (1e-3, 1.0, 4e3, 0.0), (1e-12, 1e12)])
@pytest.mark.parametrize("b,ctx,nh,nkv", [(5, 300, 4, 2), (64, 1000, 64, 1), (900, 300, 4, 2)])
def test_large_scores_of_values_of_other_sizes(ops, ws, b, ctx, nh, nkv, sizes, power):
    """The same with values of another size, row by row: the mean of the values
    of a row's largest scores, rounded by the largest of these."""
    T = ops.DevTensor
    r = np.random.default_rng(b + power)
    q, k, v = tensors(r, b, ctx, nh, nkv, "float32", extra=b)
    for t in (q, k):
        t[...] = np.where(t < 0, -1, 1)
        t[..., 6:] = 0
        t *= np.float32(2.0 ** power)
    v *= np.float32(sizes)[np.arange(ctx + b) * 7 % len(sizes)][None, :, None]
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k), T.of(v), out, ws, pos0=ctx, scale=0.125)
    got, hpk = out.numpy(), nh // nkv
    for h in range(nh):
        s = np.einsum("id,jd->ij", q[:, h], k[h // hpk])
        s[~visible(b, ctx, 0, 0)] = -np.inf
        top = s == s.max(1, keepdims=True)
        val = v[h // hpk].astype(np.float64)
        want = top @ val / top.sum(1, keepdims=True)
        most = (top * np.abs(val).max(1)).max(1, keepdims=True)
        check(got[:, h], want, most * U * (8 * np.sqrt(ctx + b) + 16))


@pytest.mark.parametrize("power", [12, 20, 30])
@pytest.mark.parametrize("b,ctx,nh,nkv,dtype", [(5, 300, 16, 8, "float32"), (9, 300, 16, 8, "bfloat16"),
                                                (700, 900, 16, 4, "float32"), (700, 900, 16, 4, "bfloat16")])
def test_large_scores_beside_garbage(ops, ws, b, ctx, nh, nkv, dtype, power):
    """The same, where the last row's value is infinite: keys beside it are gone
    through one by one."""
    T = ops.DevTensor
    r = np.random.default_rng(b + ctx + power)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype, extra=b)
    for t in (q, k):
        t[...] = np.where(t < 0, -1, 1)
        t[..., 6:] = 0
        t *= np.float32(2.0 ** power)
    want, tol = reference(q, k, v, visible(b, ctx, 0, 0), 0.125)
    tol = np.abs(v).max() * U * (8 * np.sqrt(ctx + b) + 16) + 0 * tol
    v[:, ctx + b - 1] = np.inf
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx, scale=0.125)
    check(out.numpy()[:-1], want[:-1], tol[:-1])


# ---- keys -----------------------------------------------------------------
@pytest.mark.parametrize("dtype,big", [("float32", 1e4), ("float32", 1e6), ("float32", 1e10), ("float32", 1e30),
                                       ("float16", 1e4), ("bfloat16", 1e6), ("bfloat16", 1e30)])
@pytest.mark.parametrize("b,nh,nkv,ctx,window", [(5, 16, 4, 300, 280), (64, 16, 4, 300, 280), (64, 64, 1, 1300, 1280)])
def test_keys_of_another_size_seen_by_some_rows(ops, ws, b, nh, nkv, ctx, window, dtype, big):
    """A leaf of a tree, and a cached position that only the first rows see
    through their window, hold keys `big` times the others."""
    r = np.random.default_rng(21)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype)
    _, kn, vn = tensors(r, b, b, nh, nkv, dtype)
    mask, depth = ops.tree_masks([-1] + [max(0, i - 2) for i in range(1, b)], pos0=ctx, window=window)
    near = np.float32(1 if dtype == "float16" else 4)  # (f16 ends at 65504)
    for t, at in ((k, ctx - window + 1), (kn, b - 1)):
        t[:, at] = rounded(np.clip(t[:, at], -near, near) * np.float32(big), dtype)
    see = visible(b, ctx, window, 0, mask, depth)
    want, tol = reference(q, np.concatenate([k, kn], 1), np.concatenate([v, vn], 1), see)
    check(run_tree(ops, ws, q, k, v, kn, vn, dtype, ctx, mask, depth, window), want, tol)


@pytest.mark.parametrize("small", [1e-4, 1e-12])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("b", [100, 2000])
def test_small_keys_between_ordinary_ones(ops, ws, b, small, dtype):
    """Through a window of two, half the rows see keys `small` times the ordinary
    ones beside them, with queries as much larger: scores of the usual size."""
    T = ops.DevTensor
    r = np.random.default_rng(22)
    q, k, v = tensors(r, b, 0, 16, 8, dtype, extra=b)
    at = np.arange(b) % 4
    k[:, at != 1] = rounded(k[:, at != 1] * np.float32(small), dtype)
    q[(at == 0) | (at == 3)] /= np.float32(small)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, window=2)
    check(out.numpy(), *reference(q, k, v, visible(b, 0, 2, 0)))


@pytest.mark.parametrize("dtype,big", [("float32", 1e4), ("float32", 1e6), ("float32", 1e12), ("float16", 1e4),
                                       ("bfloat16", 1e6)])
@pytest.mark.parametrize("b,window", [(200, 30), (1600, 1000)])
def test_large_keys_in_a_chunk(ops, ws, b, window, dtype, big):
    """The rows before the middle of a chunk do not see its far larger key."""
    T = ops.DevTensor
    r = np.random.default_rng(23)
    q, k, v = tensors(r, b, 0, 16, 8, dtype, extra=b)
    k[:, b // 2] = rounded(np.clip(k[:, b // 2], -4, 4) * np.float32(big), dtype)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, window=window)
    check(out.numpy(), *reference(q, k, v, visible(b, 0, window, 0)))


# ---- values ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("first,rest", [(1, 1e6), (1, 1e8), (1, 1e30), (1e-8, 1), (1e-12, 1), (1e-8, 1e8), (1e8, 1)])
@pytest.mark.parametrize("b", [200, 1100])
def test_a_first_value_of_another_size(ops, ws, b, first, rest, dtype):
    """Row 0 sees its own value alone, which may be far smaller than all others."""
    T = ops.DevTensor
    r = np.random.default_rng(24)
    q, k, v = tensors(r, b, 0, 16, 8, dtype, extra=b)
    v *= np.float32(rest)
    v[:, 0] *= np.float32(first / rest)
    v = rounded(v, dtype)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws)
    check(out.numpy(), *reference(q, k, v, visible(b, 0, 0, 0)))


@pytest.mark.parametrize("dtype,big", [("float32", 1e3), ("float32", 1e6), ("float32", 1e25), ("bfloat16", 1e6),
                                       ("float16", 1e4), ("float32", 1e-6), ("float32", 1e-25)])
@pytest.mark.parametrize("b,window", [(100, 1), (2000, 1), (2000, 3)])
def test_neighbours_with_values_of_another_size(ops, ws, b, window, dtype, big):
    """Every fourth row of a chunk has values `big` times the others'; the rows
    around it see it through a short window, or not at all."""
    T = ops.DevTensor
    r = np.random.default_rng(25)
    q, k, v = tensors(r, b, 0, 16, 8, dtype, extra=b)
    v[:, 1::4] = rounded(np.clip(v[:, 1::4], -4, 4) * np.float32(big), dtype)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, window=window)
    check(out.numpy(), *reference(q, k, v, visible(b, 0, window, 0)))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("b,ctx", [(5, 300), (64, 900), (700, 900)])
def test_rows_of_zeros(ops, ws, b, ctx, dtype):
    """Keys and values of zeros (a position that was never written) among
    others, and rows that see nothing but zeros."""
    T = ops.DevTensor
    r = np.random.default_rng(26)
    q, k, v = tensors(r, b, ctx, 16, 4, dtype, extra=b)
    v[:, ::3] = 0
    k[:, ::5] = 0
    v[:, :40] = k[:, :40] = 0
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx, window=ctx // 2, sinks=20)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, ctx // 2, 20)))


@pytest.mark.parametrize("std", [0.02, 1e-4, 300.0])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_values_and_keys_of_one_other_size(ops, ws, std, dtype):
    T = ops.DevTensor
    r = np.random.default_rng(27)
    b, ctx = 300, 1000
    q, k, v = tensors(r, b, ctx, 16, 4, dtype, extra=b)
    k, v = (rounded(t * np.float32(std), dtype) for t in (k, v))
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx)
    want, tol = reference(q, k, v, visible(b, ctx, 0, 0))
    check(out.numpy(), want, tol)


# ---- the ends of the range -------------------------------------------------
@pytest.mark.parametrize("size", [1e-33, 1e-30, 1e30, 1e33])
@pytest.mark.parametrize("scale", [0.0, 1e-6])
@pytest.mark.parametrize("b,ctx", [(4, 300), (64, 300), (300, 400)])
def test_far_keys(ops, ws, b, ctx, size, scale):
    """Keys of 1e33 (1e-33) against queries of 1e-33 (1e33): ordinary scores, or
    small ones with a scale of 1e-6."""
    T = ops.DevTensor
    r = np.random.default_rng(28)
    q, k, v = tensors(r, b, ctx, 8, 2, "float32", extra=b)
    q, k = q / np.float32(size), k * np.float32(size)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k), T.of(v), out, ws, pos0=ctx, scale=scale)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, 0, 0), scale or HD ** -0.5))


@pytest.mark.parametrize("b,ctx", [(4, 300), (64, 300), (1000, 400)])
def test_queries_of_1e_37(ops, ws, b, ctx):
    """and a scale that makes ordinary scores of them"""
    T = ops.DevTensor
    r = np.random.default_rng(32)
    q, k, v = tensors(r, b, ctx, 8, 2, "float32", extra=b)
    q, k = q * np.float32(1e-37), k * np.float32(1e29)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k), T.of(v), out, ws, pos0=ctx, scale=1e7)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, 0, 0), np.float32(1e7)))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [1e-33, 1e-25, 1e25, 1e33])
@pytest.mark.parametrize("b,ctx", [(4, 300), (64, 300), (300, 400)])
def test_far_values(ops, ws, b, ctx, size, dtype):
    T = ops.DevTensor
    r = np.random.default_rng(29)
    q, k, v = tensors(r, b, ctx, 8, 2, dtype, extra=b)
    v = rounded(v * np.float32(size), dtype)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, 0, 0)))


@pytest.mark.parametrize("b,ctx,nh,nkv", [(2, 300, 4, 2), (64, 300, 16, 4)])
def test_queries_at_the_end_of_the_range(ops, ws, b, ctx, nh, nkv):
    """Queries down to 1e-38 against f16 keys: every score is 0 within f32, the
    output the mean of the values."""
    T = ops.DevTensor
    r = np.random.default_rng(30)
    q, k, v = tensors(r, b, ctx, nh, nkv, "float16", extra=b)
    q *= np.float32(1e-38)
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, "float16"), T.of(v, "float16"), out, ws, pos0=ctx, scale=1e4)
    check(out.numpy(), *reference(q, k, v, visible(b, ctx, 0, 0), 1e4))


# ---- rows one by one -------------------------------------------------------
@pytest.mark.parametrize("places", [[0], [70], [0, -1], [3, 64, 1000, 2999], [63, 64, 65, 127, 128, 2000, -1]])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("b,ctx,nh,nkv", [(5, 3001, 16, 8), (64, 3001, 64, 1), (900, 2500, 16, 8)])
def test_odd_rows_here_and_there(ops, ws, b, ctx, nh, nkv, dtype, places):
    """Rows that are gone through one by one: values of 1e30 or 1e-30, keys of
    1e-33, and an infinite value that the last row alone sees."""
    T = ops.DevTensor
    r = np.random.default_rng(31)
    q, k, v = tensors(r, b, ctx, nh, nkv, dtype, extra=b)
    for i, at in enumerate(places):
        t, f = ((v, 1e-30), (k, 1e-33), (v, 1e30))[i % 3]
        t[:, at] *= np.float32(f)
    k, v = rounded(k, dtype), rounded(v, dtype)
    want, tol = reference(q, k, v, visible(b, ctx, 0, 0))
    v[:, -1] = np.inf
    out = filled(ops, q.shape)
    ops.attention(T.of(q), T.of(k, dtype), T.of(v, dtype), out, ws, pos0=ctx)
    check(out.numpy()[:-1], want[:-1], tol[:-1])


# ---- a first call that is captured ----------------------------------------
FIRST = """
import ctypes as C
import numpy as np
import cmf_amd
from cmf_amd import ops
cmf_amd.init(0)
T = ops.DevTensor
r = np.random.default_rng(1)
n, nh, nkv = 300, 16, 4
q, k, v = (T.of(r.standard_normal(s, dtype=np.float32)) for s in ((n, nh, 128), (nkv, n, 128), (nkv, n, 128)))
out, eager, ws = T.of(np.zeros((n, nh, 128), np.float32)), T.empty((n, nh, 128)), T.empty(64 << 20, "uint8")
hip = C.CDLL("libamdhip64.so.7")
ok = lambda rc: rc and exit(f"HIP error {rc}")
s, g, e = C.c_void_p(), C.c_void_p(), C.c_void_p()
cmf_amd.check(cmf_amd.lib().cmf_sync())
ok(hip.hipStreamCreateWithFlags(C.byref(s), 1))
ok(hip.hipStreamBeginCapture(s, MODE))
ops.attention(q, k, v, out, ws, stream=s.value)
ok(hip.hipStreamEndCapture(s, C.byref(g)))
ok(hip.hipGraphInstantiate(C.byref(e), g, None, None, C.c_size_t(0)))
ops.attention(q, k, v, eager, ws)
want = eager.numpy()
for i in range(3):
    out.buf.upload(np.full((n, nh, 128), 3, np.float32))
    ok(hip.hipGraphLaunch(e, s))
    ok(hip.hipStreamSynchronize(s))
    assert np.array_equal(out.numpy(), want)
print("done")
"""


@pytest.mark.parametrize("mode", [0, 1])
def test_a_first_call_may_be_captured(gpu, mode):
    """In a process that has made no call before, and in every capture mode."""
    r = subprocess.run([sys.executable, "-c", FIRST.replace("MODE", str(mode))], cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout[-300:] + r.stderr[-1500:]
