"""Device memory, streams and graph capture for tests of the entry points on caller-owned memory, through the HIP runtime
that the library itself links (already loaded with it)."""
import ctypes as C

import numpy as np

H2D, D2H = 1, 2
CAPTURE_RELAXED = 2


class Hip:
    def __init__(self, gq):
        gq.hip_lib()
        self.rt = C.CDLL("libamdhip64.so.7", mode=C.RTLD_GLOBAL)
        vp, pvp = C.c_void_p, C.POINTER(C.c_void_p)
        for name, args in (("hipMalloc", [pvp, C.c_size_t]), ("hipFree", [vp]), ("hipMemcpy", [vp, vp, C.c_size_t, C.c_int]),
                           ("hipDeviceSynchronize", []), ("hipSetDevice", [C.c_int]), ("hipStreamCreate", [pvp]),
                           ("hipStreamDestroy", [vp]), ("hipStreamSynchronize", [vp]), ("hipStreamBeginCapture", [vp, C.c_int]),
                           ("hipStreamEndCapture", [vp, pvp]), ("hipGraphInstantiate", [pvp, vp, vp, vp, C.c_size_t]),
                           ("hipGraphLaunch", [vp, vp]), ("hipGraphExecDestroy", [vp]), ("hipGraphDestroy", [vp])):
            fn = getattr(self.rt, name)
            fn.restype, fn.argtypes = C.c_int, args
        self.ok(self.rt.hipSetDevice(0))
        self.held, self.streams, self.graphs = [], [], []

    @staticmethod
    def ok(st):
        assert st == 0, f"HIP status {st}"

    def alloc(self, nbytes):
        p = C.c_void_p()
        self.ok(self.rt.hipMalloc(C.byref(p), max(int(nbytes), 256)))
        self.held.append(p.value)
        return p.value

    def upload(self, a):
        a = np.ascontiguousarray(a)
        p = self.alloc(a.nbytes)
        self.write(p, a)
        return p

    def write(self, p, a):
        a = np.ascontiguousarray(a)
        if a.nbytes:
            self.ok(self.rt.hipMemcpy(p, a.ctypes.data, a.nbytes, H2D))
            self.sync()

    def download(self, p, shape, dtype):
        self.sync()
        out = np.empty(shape, dtype)
        if out.nbytes:
            self.ok(self.rt.hipMemcpy(out.ctypes.data, p, out.nbytes, D2H))
        return out

    def sync(self):
        self.ok(self.rt.hipDeviceSynchronize())

    def stream(self):
        s = C.c_void_p()
        self.ok(self.rt.hipStreamCreate(C.byref(s)))
        self.streams.append(s.value)
        return s.value

    def capture(self, stream, work):
        """The work queued by work() on the stream, as a graph that can be launched."""
        self.ok(self.rt.hipStreamBeginCapture(stream, CAPTURE_RELAXED))
        work()
        g, x = C.c_void_p(), C.c_void_p()
        self.ok(self.rt.hipStreamEndCapture(stream, C.byref(g)))
        self.ok(self.rt.hipGraphInstantiate(C.byref(x), g, None, None, 0))
        self.graphs.append((g.value, x.value))
        return x.value

    def launch(self, graph, stream):
        self.ok(self.rt.hipGraphLaunch(graph, stream))

    def close(self):
        self.rt.hipDeviceSynchronize()
        for g, x in self.graphs:
            self.rt.hipGraphExecDestroy(x)
            self.rt.hipGraphDestroy(g)
        for s in self.streams:
            self.rt.hipStreamDestroy(s)
        for p in self.held:
            self.rt.hipFree(p)
        self.held, self.streams, self.graphs = [], [], []
