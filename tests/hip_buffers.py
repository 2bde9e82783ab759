"""Device buffers, streams and graphs for GPU tests, straight from the HIP runtime through ctypes."""
from __future__ import annotations

import ctypes as C

import numpy as np


class Hip:
    def __init__(self):
        h = self.h = C.CDLL("libamdhip64.so")
        P = C.c_void_p
        h.hipMalloc.argtypes = [C.POINTER(P), C.c_size_t]
        h.hipFree.argtypes = [P]
        h.hipMemcpy.argtypes = [P, P, C.c_size_t, C.c_int]
        h.hipStreamCreateWithFlags.argtypes = [C.POINTER(P), C.c_uint]
        h.hipStreamDestroy.argtypes = h.hipStreamSynchronize.argtypes = [P]
        h.hipStreamBeginCapture.argtypes = [P, C.c_int]
        h.hipStreamEndCapture.argtypes = [P, C.POINTER(P)]
        h.hipGraphInstantiate.argtypes = [C.POINTER(P), P, P, P, C.c_size_t]
        h.hipGraphLaunch.argtypes = [P, P]
        h.hipGraphExecDestroy.argtypes = h.hipGraphDestroy.argtypes = [P]
        self.bufs, self.streams, self.graphs = [], [], []

    def ok(self, rc):
        assert rc == 0, f"HIP error {rc}"

    def alloc(self, nbytes: int) -> int:
        p = C.c_void_p()
        self.ok(self.h.hipMalloc(C.byref(p), max(nbytes, 16)))
        self.bufs.append(p.value)
        return p.value

    def write(self, p: int, a: np.ndarray):
        a = np.ascontiguousarray(a)
        self.ok(self.h.hipMemcpy(p, a.ctypes.data, a.nbytes, 1))

    def put(self, a: np.ndarray) -> int:
        p = self.alloc(a.nbytes)
        self.write(p, a)
        return p

    def get(self, p: int, like: np.ndarray) -> np.ndarray:
        out = np.empty_like(like)
        self.sync()
        self.ok(self.h.hipMemcpy(out.ctypes.data, p, out.nbytes, 2))
        return out

    def sync(self):
        self.ok(self.h.hipDeviceSynchronize())

    def stream(self) -> int:
        p = C.c_void_p()
        self.ok(self.h.hipStreamCreateWithFlags(C.byref(p), 1))   # does not wait for the default stream
        self.streams.append(p.value)
        return p.value

    def capture(self, stream: int, work) -> int:
        """The executable graph of what work() enqueues on the stream."""
        self.ok(self.h.hipStreamBeginCapture(stream, 1))   # thread-local
        work()
        g, e = C.c_void_p(), C.c_void_p()
        self.ok(self.h.hipStreamEndCapture(stream, C.byref(g)))
        self.ok(self.h.hipGraphInstantiate(C.byref(e), g, None, None, 0))
        self.graphs.append((g.value, e.value))
        return e.value

    def launch(self, graph: int, stream: int):
        self.ok(self.h.hipGraphLaunch(graph, stream))

    def close(self):
        self.sync()
        for g, e in self.graphs:
            self.h.hipGraphExecDestroy(e)
            self.h.hipGraphDestroy(g)
        for s in self.streams:
            self.h.hipStreamDestroy(s)
        for p in self.bufs:
            self.h.hipFree(p)
        self.bufs, self.streams, self.graphs = [], [], []
