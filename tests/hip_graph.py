"""A HIP graph captured from the library's launches, by the runtime that it
is linked to."""
import ctypes

_hip = None


def _call(name, *args):
    global _hip
    if _hip is None:
        _hip = ctypes.CDLL("/opt/rocm/lib/libamdhip64.so")
    rc = getattr(_hip, name)(*args)
    assert rc == 0, (name, rc)


class Graph:
    """Captures what body() launches on stream (a Stream of phobos_amd)."""

    def __init__(self, stream, body):
        self.stream = ctypes.c_void_p(stream.handle)
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        _call("hipStreamBeginCapture", self.stream, 0)  # the strictest mode
        try:
            body()
        finally:
            _call("hipStreamEndCapture", self.stream, ctypes.byref(graph))
        _call("hipGraphInstantiate", ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0))
        _call("hipGraphDestroy", graph)

    def replay(self):
        _call("hipGraphLaunch", self.exec, self.stream)

    def destroy(self):
        _call("hipGraphExecDestroy", self.exec)
