"""Device arrays, streams and graphs for the tests, through the HIP runtime the library is linked against."""
import ctypes

import numpy as np

import speculate_hip

P = ctypes.c_void_p


def runtime():
    rt = speculate_hip._hip_runtime()
    if not getattr(rt, "_tests", False):
        rt.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(P), ctypes.c_uint]
        for name in ("hipStreamSynchronize", "hipStreamDestroy", "hipGraphExecDestroy", "hipGraphDestroy"):
            getattr(rt, name).argtypes = [P]
        rt.hipStreamBeginCapture.argtypes = [P, ctypes.c_int]
        rt.hipStreamEndCapture.argtypes = [P, ctypes.POINTER(P)]
        rt.hipGraphInstantiate.argtypes = [ctypes.POINTER(P), P, P, P, ctypes.c_size_t]
        rt.hipGraphLaunch.argtypes = [P, P]
        rt._tests = True
    return rt


def check(code):
    assert code == 0, f"HIP error {code}"


def synchronize():
    check(runtime().hipDeviceSynchronize())


class Dev:
    """A device array; freed with the object."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape if isinstance(shape, tuple) else (shape,), np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        self._p = P()
        check(runtime().hipMalloc(ctypes.byref(self._p), max(self.nbytes, 16)))

    @property
    def ptr(self):
        return int(self._p.value)

    def put(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        assert a.nbytes == self.nbytes
        if a.nbytes:
            check(runtime().hipMemcpy(self._p, a.ctypes.data_as(P), a.nbytes, 1))
            synchronize()
        return self

    def get(self):
        out = np.empty(self.shape, self.dtype)
        synchronize()
        if out.nbytes:
            check(runtime().hipMemcpy(out.ctypes.data_as(P), self._p, out.nbytes, 2))
        return out

    def __del__(self):
        try:
            runtime().hipFree(self._p)
        except Exception:
            pass


def dev(a):
    a = np.asarray(a)
    return Dev(a.shape, a.dtype).put(a)


def full(shape, value, dtype=np.float32):
    return dev(np.full(shape, value, dtype))


def zeros(shape, dtype=np.float32):
    return full(shape, 0, dtype)


def ptr(d):
    return 0 if d is None else d.ptr


class Stream:
    """A stream of its own (non-blocking)."""

    def __init__(self):
        self._s = P()
        check(runtime().hipStreamCreateWithFlags(ctypes.byref(self._s), 1))

    @property
    def handle(self):
        return int(self._s.value)

    def wait(self):
        check(runtime().hipStreamSynchronize(self._s))

    def __del__(self):
        try:
            runtime().hipStreamDestroy(self._s)
        except Exception:
            pass


class Graph:
    """step(stream handle) recorded once; launch() replays it and waits."""

    def __init__(self, step):
        rt, self.stream = runtime(), Stream()
        graph, self._ex = P(), P()
        check(rt.hipStreamBeginCapture(self.stream._s, 0))
        try:
            step(self.stream.handle)
        finally:
            rc = rt.hipStreamEndCapture(self.stream._s, ctypes.byref(graph))
        check(rc)
        check(rt.hipGraphInstantiate(ctypes.byref(self._ex), graph, None, None, 0))
        check(rt.hipGraphDestroy(graph))

    def launch(self):
        check(runtime().hipGraphLaunch(self._ex, self.stream._s))
        self.stream.wait()

    def __del__(self):
        try:
            runtime().hipGraphExecDestroy(self._ex)
        except Exception:
            pass
