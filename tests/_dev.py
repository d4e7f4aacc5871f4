"""Device arrays for the tests of the attention entry points: the HIP runtime that libatlas_hip.so links (torch brings one of its own, which cannot open the
device once another has), numpy on the host side."""
import ctypes as C

import numpy as np

_hip = None


def hip():
    global _hip
    if _hip is None:
        import jolt_atlas_amd  # noqa: F401  (maps the runtime)
        _hip = C.CDLL("libamdhip64.so.7")
    return _hip


def ok(rc):
    assert rc == 0, f"HIP error {rc}"


class Buffer:
    def __init__(self, n):
        self.p = C.c_void_p()
        ok(hip().hipMalloc(C.byref(self.p), C.c_size_t(max(n, 16))))

    def __del__(self):
        if _hip is not None and self.p:
            _hip.hipFree(self.p)


class Dev:
    """a view of device memory: what jolt_atlas_amd.attention asks of a tensor, and the way back to numpy"""

    def __init__(self, host, buf=None, at=0, shape=None, strides=None):
        if buf is None:
            host = np.ascontiguousarray(host)
            buf = Buffer(host.nbytes)
            if host.nbytes:
                ok(hip().hipMemcpy(buf.p, host.ctypes.data_as(C.c_void_p), C.c_size_t(host.nbytes), C.c_int(1)))
            shape, strides = host.shape, tuple(s // host.itemsize for s in host.strides)
            self.total = host.size
        self.buf, self.at, self.shape, self._strides, self.dtype = buf, at, tuple(shape), tuple(strides), np.dtype(host.dtype)
        self.itemsize = self.dtype.itemsize

    def data_ptr(self):
        return self.buf.p.value + self.at * self.itemsize

    def stride(self):
        return self._strides

    def view(self, at, shape, strides):
        v = Dev(np.empty(0, self.dtype), self.buf, self.at + at, shape, strides)
        v.total = self.total
        return v

    def numpy(self):
        """the whole buffer as it is now (a view gives its own elements)"""
        ok(hip().hipDeviceSynchronize())
        flat = np.empty(self.total, self.dtype)
        if flat.nbytes:
            ok(hip().hipMemcpy(flat.ctypes.data_as(C.c_void_p), self.buf.p, C.c_size_t(flat.nbytes), C.c_int(2)))
        return np.lib.stride_tricks.as_strided(flat[self.at:], self.shape, [s * self.itemsize for s in self._strides]).copy()


def workspace(n):
    """n bytes of device memory that hold anything but zeros"""
    b = Buffer(n)
    ok(hip().hipMemset(b.p, C.c_int(0xA5), C.c_size_t(max(n, 16))))
    ok(hip().hipDeviceSynchronize())
    v = Dev(np.empty(0, np.uint8), b, 0, (max(n, 16),), (1,))
    v.total = max(n, 16)
    return v
