"""What a call of cmf_attention_dev is planned for, by the scratch it asks for
(cmf_attention_workspace), on the CPU."""
import ctypes as C

import pytest

import cmf_amd
from test_ops_refusals import X, attn


def workspace(**kw):
    return cmf_amd.lib().cmf_attention_workspace(C.byref(attn(nh=16, nkv=8, ldq=2048, ldo=2048, slots=1 << 20, **kw)))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("b", [1, 5, 17, 100, 512, 700, 1000, 2048])
@pytest.mark.parametrize("pos0", [0, 1, 100, 5000])
@pytest.mark.parametrize("window,sinks", [(0, 0), (400, 0), (900, 4), (5000, 0)])
def test_a_position_on_the_device_is_planned_for_as_one_on_the_host(b, pos0, window, sinks, dtype):
    """with a bound that equals the position: a chunk's rows are keys of its own"""
    kw = dict(b=b, window=window, sinks=sinks, kv_dtype=dtype)
    assert workspace(pos0=0, d_pos0=X, len_bound=pos0, **kw) == workspace(pos0=pos0, **kw)
