"""Operators on device tensors around the verification of drafted tokens
(libcmfhip cmf_*_dev): head norms with the rotation, attention of a token tree
or through a sliding window over a cache, copies of cache rows, and log
probabilities.

The functions take device tensors by their pointers: anything with data_ptr(),
shape, stride() and dtype, as DevTensor below or torch tensors (a process that
uses torch on the GPU imports it before this library is loaded: both bring a
HIP runtime, and the first one serves both).  They lie on the library's device
(cmf_init's, else 0): a tensor whose get_device() says otherwise is refused.
Head rows have 128 elements and are contiguous; activations are f32, caches and
logits f32, f16 or bf16.  Nothing is allocated, checked on the device or waited
for; outputs are written in place.  stream: None for the calling thread's
library stream (cmf_amd.lib().cmf_sync() waits for it), or a HIP stream handle
(torch: stream.cuda_stream; 0 is the null stream).  The library's stream waits
for no other one: tensors that torch's work still reads or writes go with
torch's stream.  Raises CmfError when the library refuses the arguments.
"""
import ctypes as C
import struct

import numpy as np

from . import AttentionArgs, CmfError, DevBuf, KvCopyArgs, LogprobsArgs, QkRopeArgs, _ptr, check, lib

DT_F32, DT_F16, DT_BF16 = 0, 1, 2
_DTYPES = {"float32": DT_F32, "float16": DT_F16, "bfloat16": DT_BF16}
STREAM_NULL = 1  # CMF_STREAM_NULL
WORKSPACE_MAX = 64 << 20  # no call asks for more scratch


class DevTensor:
    """A device tensor of the library: a strided view of a DevBuf."""
    SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8, "uint64": 8, "uint8": 1}

    def __init__(self, buf, shape, strides, dtype, offset=0):
        self.buf, self.shape, self._strides, self.dtype, self.offset = buf, tuple(shape), tuple(strides), dtype, offset

    @classmethod
    def of(cls, array, dtype=None):
        """A numpy array on the device, as `dtype` (its own; f32 arrays also
        rounded to float16 or bfloat16)."""
        dtype = dtype or str(array.dtype)
        a = np.ascontiguousarray(array)
        if dtype == "bfloat16":
            u = a.astype(np.float32).view(np.uint32)
            up = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
            a = np.where(np.isnan(a), np.uint16(0x7fc0), up)
        else:
            a = a.astype(dtype)
        t = cls.empty(a.shape, dtype)
        if a.size:
            t.buf.upload(a)
        return t

    @classmethod
    def empty(cls, shape, dtype="float32"):
        shape = (shape,) if isinstance(shape, int) else tuple(shape)
        strides = [int(np.prod(shape[i + 1:], dtype=np.int64)) for i in range(len(shape))]
        n = int(np.prod(shape, dtype=np.int64))
        return cls(DevBuf(max(16, n * cls.SIZES[dtype])), shape, strides, dtype)

    def get_device(self):
        return _device_of_library()

    def data_ptr(self):
        return self.buf.p + self.offset * self.element_size()

    def element_size(self):
        return self.SIZES[self.dtype]

    def stride(self):
        return self._strides

    def __getitem__(self, key):
        key = key if isinstance(key, tuple) else (key,)
        if len(key) > len(self.shape):
            raise IndexError(f"{len(key)} indices for {len(self.shape)} dimensions")
        shape, strides, off = [], [], self.offset
        for i, (n, st) in enumerate(zip(self.shape, self._strides)):
            k = key[i] if i < len(key) else slice(None)
            if isinstance(k, slice):
                lo, hi, step = k.indices(n)
                off += lo * st
                shape.append(max(0, -(-(hi - lo) // step)))
                strides.append(st * step)
            else:
                if not -n <= k < n:
                    raise IndexError(f"index {k} of {n}")
                off += (k % n) * st
        return DevTensor(self.buf, shape, strides, self.dtype, off)

    def permute(self, *axes):
        return DevTensor(self.buf, [self.shape[i] for i in axes], [self._strides[i] for i in axes], self.dtype, self.offset)

    def numpy(self):
        """The values on the host (16-bit floats as f32); waits for the calling
        thread's library stream."""
        check(lib().cmf_sync())
        raw = {"bfloat16": "uint16"}.get(self.dtype, self.dtype)
        flat = self.buf.download(self.buf.nbytes // self.element_size(), raw)
        es = self.element_size()
        a = np.lib.stride_tricks.as_strided(flat[self.offset:], self.shape, [s * es for s in self._strides]).copy()
        if self.dtype == "bfloat16":
            return (a.astype(np.uint32) << 16).view(np.float32)
        return a.astype(np.float32) if self.dtype == "float16" else a


# The wrappers are on the path of every drafted token, so they read each of a
# tensor's properties once and write a message only when it is needed.
_SEEN = {}  # dtype object -> its plain name ("float32")


def _name(t):
    d = t.dtype
    try:
        return _SEEN[d]
    except KeyError:
        return _SEEN.setdefault(d, str(d).replace("torch.", ""))


def _dt(t):
    try:
        return _DTYPES[_name(t)]
    except KeyError:
        raise CmfError(f"dtype {t.dtype}: f32, f16 or bf16") from None


_device = None  # the library's, once it has one


def _device_of_library():
    global _device
    if _device is None:
        d = lib().cmf_device()
        if d < 0:
            return 0  # (what the first call will take)
        _device = d
    return _device


def _p(t):
    if t is None:
        return 0
    try:
        d = t.get_device()
    except AttributeError:  # (a pointer and a layout, no more)
        return t.data_ptr()
    if d != _device and d != _device_of_library():
        raise CmfError(f"a tensor {'of device %d' % d if d >= 0 else 'on the host'}: the library's device is "
                       f"{_device_of_library()}")
    return t.data_ptr()


def _stream(s):
    return 0 if s is None else (s or STREAM_NULL)


class _Call:
    """A library function of one argument struct, called with the struct's
    fields: packed in one go, which a ctypes struct takes 1 us longer for."""
    CODES = {C.c_void_p: "P", C.c_size_t: "N", C.c_longlong: "q", C.c_int: "i", C.c_double: "d", C.c_float: "f"}

    def __init__(self, name, args, result=C.c_int):
        self.name, self.result, self.fn = name, result, None
        layout = struct.Struct("".join(self.CODES[t] for _, t in args._fields_))
        assert layout.size == C.sizeof(args), name
        self.pack = layout.pack

    def __call__(self, fields):
        if self.fn is None:
            at = C.cast(getattr(lib(), self.name), C.c_void_p).value
            self.fn = C.CFUNCTYPE(self.result, C.c_char_p)(at)
        try:
            a = self.pack(*fields)
        except (struct.error, OverflowError) as e:
            raise CmfError(f"{self.name}: {e}") from None
        return self.fn(a)


_qk_rope = _Call("cmf_qk_rope_dev", QkRopeArgs)
_attention = _Call("cmf_attention_dev", AttentionArgs)
_attention_ws = _Call("cmf_attention_workspace", AttentionArgs, C.c_size_t)
_kv_copy = _Call("cmf_kv_copy_dev", KvCopyArgs)
_logprobs = _Call("cmf_logprobs_dev", LogprobsArgs)
_logprobs_ws = _Call("cmf_logprobs_workspace", LogprobsArgs, C.c_size_t)


def _f32(t, what):
    if _name(t) != "float32":
        raise CmfError(f"{what} must be f32")


def _vector(t, n):
    """Whether t holds n elements in a row (one: without a dimension, too)."""
    shape = t.shape
    return n <= shape[0] and (t.stride()[0] == 1 or shape[0] == 1) if len(shape) == 1 else n <= 1 and not len(shape)


def _i32(t, n, what):
    if not (_name(t) == "int32" and _vector(t, n)):
        raise CmfError(f"{what} must be int32, one-dimensional and contiguous, of at least {n}")


def _cache(k, v, what):
    """k and v [nkv][slots][128] of one layout -> (nkv, slots, head, row)."""
    shape, st = k.shape, k.stride()
    if not (len(shape) == 3 and shape[2] == 128 and st[2] == 1):
        raise CmfError(f"{what} must be [heads][rows][128]")
    if v is not k and not (v.shape == shape and v.stride() == st and v.dtype == k.dtype):
        raise CmfError(f"{what}: k and v differ in layout")
    return shape[0], shape[1], st[0], st[1]


def _rows(t, what):
    """t [b][heads][128] -> (b, heads, ld)."""
    shape, st = t.shape, t.stride()
    if not (len(shape) == 3 and shape[2] == 128 and st[2] == 1 and (shape[1] == 1 or st[1] == 128)):
        raise CmfError(f"{what} must be [rows][heads][128] with contiguous heads")
    b, h, _ = shape
    return b, h, st[0] if b > 1 else max(st[0], h * 128)


def qk_rope(qkv, q, k, v, q_norm, k_norm, rope, *, pos0=0, pos0_dev=None, depth=None, at_pos=True, eps=1e-6, stream=None):
    """cmf_qk_rope_dev: qkv [b][nh + 2 nkv][128], q [b][nh][128], k / v
    [nkv][slots][128], rope [positions][64][2] (cos, sin).  Row i at position
    pos0 + depth[i] (depth None: i; pos0_dev: an int32 tensor whose value is
    added); its key and value go to row pos0 + i, or row i with
    at_pos=False.  q None: keys and values only; k and v None: queries only."""
    b, hs, ldq = _rows(qkv, "qkv")
    if (q is None and k is None) or (k is None) != (v is None):
        raise CmfError("q, or k and v")
    f32, bq, ldo, slots, hst, rst = qkv.dtype, b, 0, 0, 0, 0
    if k is not None:
        nkv, slots, hst, rst = _cache(k, v, "k / v")
    if q is not None:
        bq, nh, ldo = _rows(q, "q")
    if q is None:
        nh = hs - 2 * nkv
    elif k is None:
        nkv = (hs - nh) // 2
    if not (bq == b and hs == nh + 2 * nkv and nh > 0 and nkv > 0):
        raise CmfError("qkv must hold nh + 2 nkv heads of every row of q")
    if _name(qkv) != "float32" or (q is not None and q.dtype != f32) or rope.dtype != f32:
        raise CmfError("qkv, q and rope must be f32")
    for t in (q_norm, k_norm):
        if t is not None and not (t.dtype == f32 and t.shape == (128,) and t.stride()[0] == 1):
            raise CmfError("the norms must be f32, [128]")
    positions, *pairs = rope.shape
    if pairs != [64, 2] or rope.stride() != (128, 2, 1):
        raise CmfError("rope must be [positions][64][2], contiguous")
    if depth is not None:
        _i32(depth, b, "depth")
    if pos0_dev is not None:
        _i32(pos0_dev, 1, "pos0_dev")
    check(_qk_rope((_p(qkv), _p(q), _p(k), _p(v), _p(q_norm), _p(k_norm), _p(rope), _p(pos0_dev), _p(depth), eps, hst, rst,
                    b, nh, nkv, ldq, ldo, 0 if k is None else _dt(k), positions, pos0, slots, 1 if at_pos else 0, _stream(stream))))


def _attention_args(q, k, v, out, ws, pos0, k_new, v_new, mask, depth, window, sinks, scale, pos0_dev, len_bound, stream):
    b, nh, ldq = _rows(q, "q")
    nkv, slots, hst, rst = _cache(k, v, "k / v")
    if nkv < 1 or nh % nkv:
        raise CmfError("the query heads must be a multiple of the kv heads")
    _f32(q, "q")
    ldo = nh * 128
    if out is not None:
        bo, ho, ldo = _rows(out, "out")
        if bo != b or ho != nh or out.dtype != q.dtype:
            raise CmfError("out must be shaped as q, f32")
    nhst = nrst = 0
    if k_new is not None:
        nk, rows, nhst, nrst = _cache(k_new, v_new, "k_new / v_new")
        if nk != nkv or rows < b or k_new.dtype != k.dtype:
            raise CmfError("k_new / v_new must hold b rows of k's type")
    if mask is not None and not (_name(mask) in ("int64", "uint64") and _vector(mask, b)):
        raise CmfError("mask must be [b] of 64 bits")
    if depth is not None:
        _i32(depth, b, "depth")
    if pos0_dev is not None:
        _i32(pos0_dev, 1, "pos0_dev")
    nb = 0 if ws is None else ws.shape[0] * ws.element_size()
    return (_p(q), _p(out), _p(k), _p(v), _p(k_new), _p(v_new), _p(mask), _p(pos0_dev), _p(depth), _p(ws), nb, hst, rst, nhst,
            nrst, b, nh, nkv, ldq, ldo, _dt(k), pos0, slots, len_bound, window, sinks, scale, _stream(stream))


def attention_workspace(q, k, v, *, pos0=0, k_new=None, v_new=None, mask=None, depth=None, window=0, sinks=0,
                        pos0_dev=None, len_bound=0):
    """cmf_attention_workspace: bytes of scratch the call of these arguments
    needs (never more than WORKSPACE_MAX)."""
    return _attention_ws(_attention_args(q, k, v, None, None, pos0, k_new, v_new, mask, depth, window, sinks, 0.0, pos0_dev,
                                         len_bound, None))


def attention(q, k, v, out, ws, *, pos0=0, k_new=None, v_new=None, mask=None, depth=None, window=0, sinks=0, scale=0.0,
              pos0_dev=None, len_bound=0, stream=None):
    """cmf_attention_dev: q and out [b][nh][128]; k / v [nkv][slots][128] hold
    pos0 cached positions; the rows' own keys and values are k_new / v_new
    [nkv][>= b][128], or the cache's rows pos0 .. pos0 + b.  mask (int64 bits,
    with depth under a window): a tree's visible new rows (tree_masks); without
    it row i sees the rows up to its own.  window, sinks: only the last window
    positions and the first sinks are seen (window 0: all).  ws: 1-d scratch
    tensor of attention_workspace bytes (None: nothing)."""
    check(_attention(_attention_args(q, k, v, out, ws, pos0, k_new, v_new, mask, depth, window, sinks, scale, pos0_dev,
                                     len_bound, stream)))


def tree_masks(parents, pos0=0, window=0, sinks=0):
    """cmf_tree_masks: (mask uint64 [b], depth int32 [b]) of the tree whose row
    i has the earlier row parents[i] as its parent (-1: a root)."""
    p = np.ascontiguousarray(parents, dtype=np.int32)
    m, d = np.empty(len(p), np.uint64), np.empty(len(p), np.int32)
    check(lib().cmf_tree_masks(_ptr(p), len(p), pos0, window, sinks, _ptr(m), _ptr(d)))
    return m, d


def kv_copy(dst_ptrs, src_ptrs, dst, src, *, n, pos0=0, idx=None, n_dev=None, pos0_dev=None, stream=None):
    """cmf_kv_copy_dev: row pos0 + i of every buffer of dst_ptrs = row idx[i]
    (None: i) of the buffer of src_ptrs, i < n (n_dev: and < its value).
    dst_ptrs / src_ptrs: int64 device tensors of base pointers; dst / src: one
    of the buffers of each side, [nkv][slots][128], for the layout."""
    nkv, ds, dh, dr = _cache(dst, dst, "dst")
    nk, ss, sh, sr = _cache(src, src, "src")
    if nk != nkv or src.dtype != dst.dtype:
        raise CmfError("dst and src must have the same heads and type")
    if _name(dst_ptrs) != "int64" or src_ptrs.dtype != dst_ptrs.dtype or dst_ptrs.stride() != (1,) or src_ptrs.stride() != (1,):
        raise CmfError("pointers must be int64, [buffers], contiguous")
    nbuf = dst_ptrs.shape[0]
    if src_ptrs.shape[0] != nbuf:
        raise CmfError("as many buffers on both sides")
    _p(dst), _p(src)  # (on the library's device, as the other buffers)
    if idx is not None:
        _i32(idx, n, "idx")
    if n_dev is not None:
        _i32(n_dev, 1, "n_dev")
    if pos0_dev is not None:
        _i32(pos0_dev, 1, "pos0_dev")
    check(_kv_copy((_p(dst_ptrs), _p(src_ptrs), _p(idx), _p(n_dev), _p(pos0_dev), dh, dr, sh, sr, nbuf, nkv,
                    _dt(dst), n, pos0, ds, ss, _stream(stream))))


def _logprobs_args(logits, target, logprob, entropy, top_ids, top_lp, top_k, ws, stream):
    shape, st = logits.shape, logits.stride()
    if len(shape) != 2 or st[1] != 1:
        raise CmfError("logits must be [rows][V]")
    rows, V = shape
    if target is not None:
        _i32(target, rows, "target")
    for t, w in ((logprob, "logprob"), (entropy, "entropy")):
        if t is not None and not (_name(t) == "float32" and _vector(t, rows)):
            raise CmfError(f"{w} must be f32, [rows]")
    for t, w, d in ((top_ids, "top_ids", "int32"), (top_lp, "top_lp", "float32")):
        if t is not None and not (_name(t) == d and len(t.shape) == 2 and t.shape[0] >= rows and t.shape[1] == top_k and
                                  t.stride() == (top_k, 1)):
            raise CmfError(f"{w} must be {d}, [rows][top_k], contiguous")
    nb = 0 if ws is None else ws.shape[0] * ws.element_size()
    return (_p(logits), _p(target), _p(logprob), _p(entropy), _p(top_ids), _p(top_lp), _p(ws), nb,
            st[0] if rows > 1 else max(st[0], V), rows, V, _dt(logits), top_k, _stream(stream))


def logprobs_workspace(logits, top_k=0):
    """cmf_logprobs_workspace: bytes of scratch for these logits."""
    return _logprobs_ws(_logprobs_args(logits, None, None, None, None, None, top_k, None, None))


def logprobs(logits, target=None, logprob=None, entropy=None, top_ids=None, top_lp=None, ws=None, *, stream=None):
    """cmf_logprobs_dev: logits [rows][V]; target int32 [rows] -> logprob f32
    [rows]; entropy f32 [rows] (nats); top_ids int32 / top_lp f32 [rows][k] the
    k most likely tokens (equal logits: the lowest id first).  Any output may be
    None.  ws: 1-d scratch tensor of logprobs_workspace bytes."""
    top = top_ids if top_ids is not None else top_lp
    check(_logprobs(_logprobs_args(logits, target, logprob, entropy, top_ids, top_lp, 0 if top is None else top.shape[1], ws,
                                   stream)))
