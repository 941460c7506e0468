"""Arguments that the operators of cmf_amd.ops refuse (before any device is
touched), and the masks of a token tree (cmf_tree_masks), both on the CPU."""
import ctypes as C

import numpy as np
import pytest

import cmf_amd
from cmf_amd import AttentionArgs, KvCopyArgs, LogprobsArgs, QkRopeArgs

X = 4096  # a pointer that is never followed


def refused(fn, args, word):
    rc = getattr(cmf_amd.lib(), fn)(C.byref(args))
    msg = cmf_amd.lib().cmf_last_error().decode()
    assert rc < 0 and word in msg, (rc, msg)


def rope(**kw):
    a = dict(qkv=X, q_out=X, k=X, v=X, q_norm=X, k_norm=X, rope=X, eps=1e-6, head_stride=128 * 64, row_stride=128, b=2, nh=4,
             nkv=2, ldq=1024, ldo=512, kv_dtype=0, max_pos=64, pos0=0, slots=64, at_pos=1)
    a.update(kw)
    return QkRopeArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(qkv=None), "null"), (dict(rope=None), "null"), (dict(q_out=None, k=None, v=None), "null"),
    (dict(k=None), "together"), (dict(b=0), "at least 1"), (dict(nh=0), "at least 1"), (dict(nkv=-1), "at least 1"),
    (dict(kv_dtype=3), "kv_dtype"), (dict(ldq=1020), "ldq"), (dict(ldq=1026), "ldq"), (dict(qkv=X + 4), "ldq"),
    (dict(ldo=508), "ldo"), (dict(rope=X + 8), "aligned"), (dict(row_stride=120), "strides"),
    (dict(row_stride=132), "strides"), (dict(head_stride=0), "overlap"), (dict(v=X + 2), "strides"),
    (dict(pos0=-1), "positions"), (dict(pos0=63), "positions"), (dict(pos0=40, slots=41), "slots"),
    (dict(at_pos=0, slots=1), "slots"), (dict(max_pos=0), "max_pos"), (dict(slots=0), "slots"),
])
def test_qk_rope_refuses(kw, word):
    refused("cmf_qk_rope_dev", rope(**kw), word)


def attn(**kw):
    a = dict(q=X, out=X, k=X, v=X, ws=X, ws_bytes=64 << 20, head_stride=128 * 256, row_stride=128, b=2, nh=4, nkv=2, ldq=512,
             ldo=512, kv_dtype=0, pos0=100, slots=256)
    a.update(kw)
    return AttentionArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(k=None), "null"), (dict(k_new=X), "together"),
    (dict(b=0), "at least 1"), (dict(nh=3), "multiple"), (dict(b=65, d_mask=X, slots=300), "64 rows"),
    (dict(d_depth=X), "d_mask"), (dict(d_mask=X, window=5), "d_depth"), (dict(kv_dtype=15), "kv_dtype"),
    (dict(ldq=510), "ldq"), (dict(ldo=256), "ldo"), (dict(row_stride=64), "strides"), (dict(head_stride=4), "strides"),
    (dict(k_new=X, v_new=X, new_row_stride=4), "strides"), (dict(row_stride=(1 << 22) + 8), "strides"),
    (dict(k_new=X, v_new=X, new_row_stride=1 << 33, new_head_stride=1 << 40), "strides"), (dict(pos0=-1), "at least 0"), (dict(window=-1), "at least 0"),
    (dict(sinks=-2), "at least 0"), (dict(pos0=255), "slots"), (dict(d_pos0=X, len_bound=255), "len_bound"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=X + 8), "aligned"),
    (dict(b=1 << 20, slots=1 << 30), "2^19"), (dict(nh=130, nkv=2, ldq=130 * 128, ldo=130 * 128), "64 query heads"), (dict(slots=(1 << 30) + 1), "2^30"),
])
def test_attention_refuses(kw, word):
    refused("cmf_attention_dev", attn(**kw), word)


def test_attention_workspace_is_bounded():
    L = cmf_amd.lib()
    for kw in (dict(), dict(b=64, nh=32, nkv=8, ldq=4096, ldo=4096, pos0=1 << 20, slots=1 << 21),
               dict(b=1, pos0=1 << 28, slots=1 << 29), dict(b=4096, pos0=4096, slots=8192),
               dict(b=300, nh=64, nkv=1, ldq=8192, ldo=8192, pos0=100000, slots=200000)):
        assert L.cmf_attention_workspace(C.byref(attn(**kw))) <= 64 << 20
    assert L.cmf_attention_workspace(C.byref(attn(b=0))) == 0


def copy(**kw):
    a = dict(d_dst=X, d_src=X, dst_head_stride=1024, dst_row_stride=128, src_head_stride=1024, src_row_stride=128, nbuf=2,
             nkv=2, n=4, pos0=0, dst_slots=8, src_slots=8)
    a.update(kw)
    return KvCopyArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(d_dst=None), "null"), (dict(d_src=None), "null"), (dict(nbuf=0), "at least 1"), (dict(nbuf=40000), "65535"),
    (dict(n=-1), "n >= 0"), (dict(kv_dtype=9), "kv_dtype"), (dict(dst_row_stride=64), "rows of 128"),
    (dict(src_head_stride=12), "multiples"), (dict(pos0=5), "dst"), (dict(pos0=-1), "dst"), (dict(src_slots=3), "src"),
    (dict(dst_head_stride=0), "overlap"),
])
def test_kv_copy_refuses(kw, word):
    refused("cmf_kv_copy_dev", copy(**kw), word)


def test_kv_copy_of_no_rows_is_done():
    assert cmf_amd.lib().cmf_kv_copy_dev(C.byref(copy(n=0))) == 0


def lp(**kw):
    a = dict(logits=X, target=X, logprob=X, entropy=X, top_ids=X, top_lp=X, ws=X, ws_bytes=64 << 20, ld=1000, rows=3, V=1000,
             dtype=0, top_k=5)
    a.update(kw)
    return LogprobsArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(logits=None), "null"), (dict(rows=0), "rows"), (dict(rows=70000), "rows"), (dict(V=0), "logits"),
    (dict(ld=999), "ld"), (dict(dtype=3), "dtype"), (dict(top_k=65), "top_k"), (dict(top_k=-1), "top_k"),
    (dict(V=4, ld=4), "top_k"), (dict(target=None), "together"), (dict(logprob=None), "together"),
    (dict(top_k=0), "top_k"), (dict(top_ids=None, top_lp=None), "top list"), (dict(logits=X + 2), "misaligned"),
    (dict(V=151936, ld=151936, ws=None), "workspace"), (dict(V=151936, ld=151936, ws_bytes=64), "workspace"),
])
def test_logprobs_refuses(kw, word):
    refused("cmf_logprobs_dev", lp(**kw), word)


def test_logprobs_workspace_is_bounded():
    L = cmf_amd.lib()
    for rows, V, k in ((1, 1 << 30, 64), (600, 1 << 20, 64), (65535, 1000, 64), (5, 151936, 8)):
        assert L.cmf_logprobs_workspace(C.byref(lp(rows=rows, V=V, ld=V, top_k=k))) <= 64 << 20


# ---- tree masks -----------------------------------------------------------
def masks_plain(parents, pos0, window, sinks):
    mask, depth = [], []
    for i in range(len(parents)):
        chain, j = [], i
        while j >= 0:
            chain.append(j)
            j = parents[j]
        depth.append(len(chain) - 1)
        mask.append(sum(1 << j for j in chain
                        if not window or depth[i] - depth[j] < window or pos0 + depth[j] < sinks))
    return mask, depth


@pytest.mark.parametrize("b", [1, 2, 9, 64])
@pytest.mark.parametrize("pos0,window,sinks", [(0, 0, 0), (100, 3, 0), (0, 2, 2), (3, 1, 5), (7, 100, 4)])
def test_tree_masks(b, pos0, window, sinks):
    from cmf_amd import ops
    r = np.random.RandomState(b)
    for parents in ([i - 1 for i in range(b)], [-1] * b, [-1] + [int(r.randint(max(-1, i - 5), i)) for i in range(1, b)]):
        m, d = ops.tree_masks(parents, pos0=pos0, window=window, sinks=sinks)
        want = masks_plain(parents, pos0, window, sinks)
        assert m.tolist() == want[0] and d.tolist() == want[1]


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 5], [-2], [-1] * 65, []])
def test_tree_masks_refuses(parents):
    from cmf_amd import ops
    with pytest.raises(cmf_amd.CmfError):
        ops.tree_masks(parents)
