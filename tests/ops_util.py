"""Helpers of the operator tests: host arrays as the storage types hold them,
and calls captured into a HIP graph on a stream of their own."""
import ctypes as C

import numpy as np


def rounded(x, dtype):
    """f32 values as dtype stores them (nearest, ties to even)."""
    x = np.asarray(x, np.float32)
    if dtype == "bfloat16":
        u = x.view(np.uint32)
        return ((u + 0x7fff + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return x.astype(dtype).astype(np.float32)


class Stream:
    """A HIP stream, and what is captured on it."""

    def __init__(self):
        self.hip = C.CDLL("libamdhip64.so.7")
        self.s, self.exec = C.c_void_p(), None
        self._ok(self.hip.hipStreamCreateWithFlags(C.byref(self.s), 1))  # hipStreamNonBlocking

    def _ok(self, rc):
        assert rc == 0, f"HIP error {rc}"

    @property
    def handle(self):
        return self.s.value

    def sync(self):
        self._ok(self.hip.hipStreamSynchronize(self.s))

    def capture(self, calls):
        g = C.c_void_p()
        self._ok(self.hip.hipStreamBeginCapture(self.s, 2))  # hipStreamCaptureModeRelaxed
        try:
            calls()
        finally:
            self._ok(self.hip.hipStreamEndCapture(self.s, C.byref(g)))
        ex = C.c_void_p()
        self._ok(self.hip.hipGraphInstantiate(C.byref(ex), g, None, None, C.c_size_t(0)))
        self._ok(self.hip.hipGraphDestroy(g))
        return ex

    def replay(self, ex):
        self._ok(self.hip.hipGraphLaunch(ex, self.s))
        self.sync()

    def drop(self, *execs):
        for e in execs:
            self._ok(self.hip.hipGraphExecDestroy(e))
        self._ok(self.hip.hipStreamDestroy(self.s))
