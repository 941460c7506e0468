"""cmf_amd.ops.qk_rope of queries alone and of keys and values alone: the rows
of a call with both."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,nh,nkv,dtype", [(1, 16, 8, "float32"), (9, 4, 1, "bfloat16"), (300, 12, 4, "float16")])
def test_one_side(gpu, b, nh, nkv, dtype):
    from cmf_amd import ops
    T = ops.DevTensor
    r = np.random.default_rng(b)
    rand = lambda *s: r.standard_normal(s, dtype=np.float32)  # noqa: E731
    x, qn, kn, tab = T.of(rand(b, nh + 2 * nkv, 128)), T.of(rand(128)), T.of(rand(128)), T.of(rand(b + 7, 64, 2))
    nines = lambda *s, dt="float32": T.of(np.full(s, 9, np.float32), dt)  # noqa: E731
    caches = [nines(nkv, b + 10, 128, dt=dtype) for _ in range(4)]
    q, q1 = nines(b, nh, 128), nines(b, nh, 128)
    ops.qk_rope(x, q, caches[0], caches[1], qn, kn, tab, pos0=7)
    ops.qk_rope(x, q1, None, None, qn, None, tab, pos0=7)
    ops.qk_rope(x, None, caches[2], caches[3], None, kn, tab, pos0=7)
    assert np.array_equal(q.numpy(), q1.numpy()) and not (q1.numpy() == 9).all()
    for one, both in ((2, 0), (3, 1)):
        assert np.array_equal(caches[one].numpy(), caches[both].numpy())
