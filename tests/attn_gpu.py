"""CPU tensors to device buffers and back, and HIP streams and graphs, for the
attention tests: one HIP runtime a process, the library's."""
import ctypes as C

import torch

from vdamd import lib


class Dev:
    """A contiguous CPU tensor's copy on the device; at(i) the address of element i."""

    def __init__(self, t):
        self.dtype, self.shape = t.dtype, tuple(t.shape)
        t = t.detach().contiguous()
        self.buf = lib.DeviceBuffer(t.numel() * t.element_size())
        self.put(t)

    @property
    def ptr(self):
        return self.buf.ptr

    def at(self, i):
        return self.buf.ptr + i * torch.empty(0, dtype=self.dtype).element_size()

    def put(self, t):
        t = t.contiguous()
        assert t.dtype == self.dtype and tuple(t.shape) == self.shape
        if t.numel():
            lib.check(lib.lib().vdk_memcpy_h2d(self.ptr, t.data_ptr(), t.numel() * t.element_size()))

    def get(self):
        lib.check(lib.lib().vdk_synchronize())
        t = torch.empty(self.shape, dtype=self.dtype)
        if t.numel():
            lib.check(lib.lib().vdk_memcpy_d2h(t.data_ptr(), self.ptr, t.numel() * t.element_size()))
        return t


def full(shape, value, dtype=torch.float32):
    return Dev(torch.full(shape, value, dtype=dtype))


def bits(t):
    """A tensor's bits, for comparisons that NaN takes part in."""
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


class Stream:
    """A HIP stream of the default priority; capture(f) records f into a graph and returns its launch."""

    def __init__(self):
        L = self.L = lib.lib()
        for name, n in (("hipStreamCreate", 1), ("hipStreamSynchronize", 1), ("hipStreamEndCapture", 2), ("hipGraphLaunch", 2)):
            getattr(L, name).argtypes = [C.c_void_p] * n
        L.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
        L.hipGraphInstantiate.argtypes = [C.c_void_p] * 4 + [C.c_size_t]
        self.ptr = C.c_void_p()
        assert L.hipStreamCreate(C.byref(self.ptr)) == 0

    def synchronize(self):
        assert self.L.hipStreamSynchronize(self.ptr) == 0

    def capture(self, f):
        graph, ex = C.c_void_p(), C.c_void_p()
        assert self.L.hipStreamBeginCapture(self.ptr, 1) == 0   # thread-local
        f(self.ptr)
        assert self.L.hipStreamEndCapture(self.ptr, C.byref(graph)) == 0
        assert self.L.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0

        def launch():
            assert self.L.hipGraphLaunch(ex, self.ptr) == 0
        return launch
