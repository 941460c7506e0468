"""The device that is current on a calling thread, around an operator's call."""
import ctypes as C
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("other", [0, 1])
def test_the_current_device_stays(gpu, other):
    """A thread's first call and its second; with one device, that one."""
    from cmf_amd import ops
    if other >= gpu.device_count():
        pytest.skip("one device")
    T = ops.DevTensor
    r = np.random.default_rng(1)
    x, out = T.of(r.standard_normal((2, 1000), dtype=np.float32)), T.empty(2)
    hip, seen = C.CDLL("libamdhip64.so.7"), []

    def calls():
        dev = C.c_int(-1)
        assert hip.hipSetDevice(other) == 0
        for _ in range(2):
            ops.logprobs(x, entropy=out)
            assert hip.hipGetDevice(C.byref(dev)) == 0
            seen.append(dev.value)
        gpu.check(gpu.lib().cmf_sync())
    t = threading.Thread(target=calls)
    t.start()
    t.join()
    assert seen == [other, other]
