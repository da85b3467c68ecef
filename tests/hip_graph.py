"""Graph capture for the tests, through the HIP runtime that the library itself is linked to."""

import ctypes as C

P = C.c_void_p


class Graph:
    """Captures what call(stream handle) enqueues; launch(stream handle) replays it."""

    def __init__(self, lib, stream, call):
        self.lib = lib
        for name, args in (("hipStreamBeginCapture", [P, C.c_int]), ("hipStreamEndCapture", [P, C.POINTER(P)]),
                           ("hipGraphInstantiate", [C.POINTER(P), P, P, P, C.c_size_t]), ("hipGraphLaunch", [P, P]),
                           ("hipGraphExecDestroy", [P]), ("hipGraphDestroy", [P])):
            getattr(lib, name).argtypes = args
        graph, self.exec = P(), P()
        self.check(lib.hipStreamBeginCapture(stream, 1))  # thread local
        try:
            call(stream)
        finally:
            self.check(lib.hipStreamEndCapture(stream, C.byref(graph)))
        self.check(lib.hipGraphInstantiate(C.byref(self.exec), graph, None, None, 0))
        self.check(lib.hipGraphDestroy(graph))

    @staticmethod
    def check(rc):
        assert rc == 0, f"HIP error {rc}"

    def launch(self, stream):
        self.check(self.lib.hipGraphLaunch(self.exec, stream))

    def close(self):
        self.check(self.lib.hipGraphExecDestroy(self.exec))
