"""What cmf_amd.ops takes for a tensor, before any device is touched: layouts and
devices by stand-ins that hold no memory."""
import pytest

import cmf_amd
from cmf_amd import ops


class Tensor:
    """A contiguous tensor that says where it lies, at a pointer that is never
    followed."""

    def __init__(self, *shape, dtype="float32", device=0, strides=None):
        self.shape, self.dtype, self.device = shape, dtype, device
        st, n = [], 1
        for s in reversed(shape):
            st.insert(0, n)
            n *= s
        self.strides = tuple(strides or st)

    def data_ptr(self):
        return 4096

    def stride(self):
        return self.strides

    def element_size(self):
        return {"float32": 4, "uint8": 1}.get(self.dtype, 8)

    def get_device(self):
        return self.device


def rope(where):
    t = {n: Tensor(*s) for n, s in dict(qkv=(2, 8, 128), q=(2, 4, 128), k=(2, 16, 128), v=(2, 16, 128), q_norm=(128,),
                                        k_norm=(128,), rope=(64, 64, 2)).items()}
    t.update(depth=Tensor(2, dtype="int32"), pos0_dev=Tensor(1, dtype="int32"))
    return ops.qk_rope, t, where


def attention(where):
    t = {n: Tensor(*s) for n, s in dict(q=(2, 4, 128), k=(2, 16, 128), v=(2, 16, 128), out=(2, 4, 128), k_new=(2, 2, 128),
                                        v_new=(2, 2, 128)).items()}
    t.update(ws=Tensor(64, dtype="uint8"), mask=Tensor(2, dtype="int64"), depth=Tensor(2, dtype="int32"),
             pos0_dev=Tensor(1, dtype="int32"))
    return ops.attention, t, where


def copy(where):
    t = dict(dst=Tensor(2, 16, 128), src=Tensor(2, 16, 128))
    t.update({n: Tensor(3, dtype="int64") for n in ("dst_ptrs", "src_ptrs")})
    t.update({n: Tensor(4, dtype="int32") for n in ("idx", "n_dev", "pos0_dev")}, n=4)
    return ops.kv_copy, t, where


def scores(where):
    t = dict(logits=Tensor(3, 100), target=Tensor(3, dtype="int32"), logprob=Tensor(3), entropy=Tensor(3),
             top_ids=Tensor(3, 5, dtype="int32"), top_lp=Tensor(3, 5), ws=Tensor(64, dtype="uint8"))
    return ops.logprobs, t, where


CALLS = [f(n) for f, names in (
    (rope, "qkv q k v q_norm k_norm rope depth pos0_dev"), (attention, "q k v out k_new v_new ws mask depth pos0_dev"),
    (copy, "dst src dst_ptrs src_ptrs idx n_dev pos0_dev"), (scores, "logits target logprob entropy top_ids top_lp ws"),
) for n in names.split()]


@pytest.mark.parametrize("device,word", [(-1, "on the host"), (1, "of device 1"), (7, "of device 7")])
@pytest.mark.parametrize("call,tensors,name", CALLS, ids=[f"{c.__name__}-{n}" for c, _, n in CALLS])
def test_tensors_of_another_device_are_refused(call, tensors, name, device, word):
    args = dict(tensors, **{name: Tensor(*tensors[name].shape, dtype=tensors[name].dtype, device=device)})
    with pytest.raises(cmf_amd.CmfError, match=word):
        call(**args)


def test_the_workspace_of_host_tensors_is_refused():
    k = Tensor(2, 16, 128, device=-1)
    with pytest.raises(cmf_amd.CmfError, match="on the host"):
        ops.attention_workspace(Tensor(2, 4, 128), k, k, pos0=3)
    with pytest.raises(cmf_amd.CmfError, match="on the host"):
        ops.logprobs_workspace(Tensor(3, 100, device=-1))


# (a call that passes the checks of its tensors ends at the library's own: no
# depth without a mask, no target without a result)
@pytest.mark.parametrize("ok,tensor", [
    (True, Tensor(2, dtype="int32")), (True, Tensor(5, dtype="int32")), (False, Tensor(1, dtype="int32")),
    (False, Tensor(2, dtype="int64")), (False, Tensor(2, dtype="int32", strides=(2,))), (False, Tensor(2, 3, dtype="int32")),
    (False, Tensor(2, 1, dtype="int32")), (False, Tensor(dtype="int32"))])
def test_vectors(ok, tensor):
    t = attention("q")[1]
    with pytest.raises(cmf_amd.CmfError, match="d_mask" if ok else "depth must be"):
        ops.attention(t["q"], t["k"], t["v"], t["out"], t["ws"], depth=tensor)
    t = scores("logits")[1]
    with pytest.raises(cmf_amd.CmfError, match="together" if ok else "target must be"):
        ops.logprobs(Tensor(2, 100), tensor, None, t["entropy"])


@pytest.mark.parametrize("ok,tensor", [
    (True, Tensor(dtype="int32")), (True, Tensor(1, dtype="int32")), (True, Tensor(1, dtype="int32", strides=(7,))),
    (False, Tensor(0, dtype="int32")), (False, Tensor(dtype="float32")), (False, Tensor(1, 1, dtype="int32"))])
def test_a_position_on_the_device(ok, tensor):
    """one number, with a dimension or without"""
    t = attention("q")[1]
    with pytest.raises(cmf_amd.CmfError, match="len_bound past" if ok else "pos0_dev must be"):
        ops.attention(t["q"], t["k"], t["v"], t["out"], t["ws"], pos0_dev=tensor, len_bound=16)


@pytest.mark.parametrize("ok,tensor", [
    (True, Tensor(2, dtype="int64")), (True, Tensor(9, dtype="uint64")), (False, Tensor(1, dtype="int64")),
    (False, Tensor(2, 2, dtype="int64")), (False, Tensor(2, dtype="int64", strides=(2,))), (False, Tensor(2, dtype="int32"))])
def test_masks(ok, tensor):
    t = attention("q")[1]
    with pytest.raises(cmf_amd.CmfError, match="needs d_depth" if ok else "mask must be"):
        ops.attention(t["q"], t["k"], t["v"], t["out"], t["ws"], mask=tensor, window=3)


@pytest.mark.parametrize("ok,tensor", [(True, Tensor(2)), (False, Tensor(1)), (False, Tensor(2, strides=(3,))),
                                       (False, Tensor(2, 4)), (False, Tensor(2, dtype="float16"))])
def test_results(ok, tensor):
    with pytest.raises(cmf_amd.CmfError, match="together" if ok else "logprob must be"):
        ops.logprobs(Tensor(2, 100), None, tensor)


def test_an_output_over_queries_of_another_stride_is_refused():
    q = Tensor(2, 4, 128, strides=(1024, 128, 1))
    k = Tensor(2, 16, 128)
    with pytest.raises(cmf_amd.CmfError, match="ldo = ldq"):
        ops.attention(q, k, k, Tensor(2, 4, 128), None)


@pytest.mark.parametrize("q,k,v,word", [
    (None, None, None, "q, or k and v"), (Tensor(2, 4, 128), Tensor(2, 16, 128), None, "q, or k and v"),
    (Tensor(2, 4, 128), None, Tensor(2, 16, 128), "q, or k and v"), (Tensor(2, 5, 128), None, None, "qkv must hold"),
    (Tensor(2, 8, 128), None, None, "qkv must hold"), (Tensor(3, 4, 128), None, None, "qkv must hold"),
    (None, Tensor(4, 16, 128), Tensor(4, 16, 128), "qkv must hold"), (Tensor(2, 4, 128, dtype="float16"), None, None, "f32"),
    # (these are in order up to the library's own check of the positions)
    (Tensor(2, 4, 128), None, None, "positions"), (None, Tensor(2, 100, 128), Tensor(2, 100, 128), "positions"),
    (Tensor(2, 6, 128), Tensor(1, 100, 128), Tensor(1, 100, 128), "positions")])
def test_queries_or_keys_alone(q, k, v, word):
    with pytest.raises(cmf_amd.CmfError, match=word):
        ops.qk_rope(Tensor(2, 8, 128), q, k, v, None, None, Tensor(64, 64, 2), pos0=63)


def test_views_of_a_device_tensor():
    t = ops.DevTensor(None, (3, 5, 128), (640, 128, 1), "float32")
    assert t[2].offset == t[-1].offset == 1280 and t[2].shape == (5, 128)
    v = t[1:, ::2, 4]
    assert v.shape == (2, 3) and v.stride() == (640, 256) and v.offset == 644
    for key in (3, -4, (0, 5), (0, 0, 128), (0, 0, 0, 0)):
        with pytest.raises(IndexError):
            t[key]
