"""Device buffers for tests of C entries that take device pointers, in the HIP runtime that the
library itself links, each with guard bytes behind it."""
import ctypes as C

import numpy as np

import catboost_rs_amd as cb

GUARD = 256


def hip():
    cb.load()
    L = C.CDLL("/opt/rocm/lib/libamdhip64.so.7")
    L.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
    L.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    L.hipFree.argtypes = [C.c_void_p]
    return L


class Buffers:
    """with Buffers() as b: p = b.put(array); q = b.out(shape, dtype); ...; b.get(q)"""

    def __enter__(self):
        self.hip, self.blocks = hip(), {}
        return self

    def __exit__(self, *_):
        self.hip.hipDeviceSynchronize()
        for p in self.blocks:
            self.hip.hipFree(C.c_void_p(p))

    def put(self, a, fill=0xA5):
        a = np.ascontiguousarray(a)
        p = C.c_void_p()
        assert self.hip.hipMalloc(C.byref(p), a.nbytes + GUARD) == 0
        host = np.full(a.nbytes + GUARD, fill, np.uint8)
        host[:a.nbytes] = np.frombuffer(a.tobytes(), np.uint8)
        assert self.hip.hipMemcpy(p, host.ctypes.data_as(C.c_void_p), host.nbytes, 1) == 0
        self.blocks[p.value] = (a.shape, a.dtype, a.nbytes)
        return p.value

    def out(self, shape, dtype):
        a = np.empty(shape, dtype)
        a.view(np.uint8).reshape(-1)[:] = 0x5A
        return self.put(a)

    def get(self, p):
        """The block's array; the guard behind it must be as it was."""
        shape, dtype, n = self.blocks[p]
        host = np.empty(n + GUARD, np.uint8)
        assert self.hip.hipDeviceSynchronize() == 0
        assert self.hip.hipMemcpy(host.ctypes.data_as(C.c_void_p), C.c_void_p(p), host.nbytes, 2) == 0
        assert (host[n:] == 0xA5).all(), "written past the end"
        return np.frombuffer(host[:n].tobytes(), dtype).reshape(shape)
