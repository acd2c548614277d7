"""How many launches a call makes: it is captured, and the graph's nodes are counted."""
import ctypes

import baloon_amd as bx


def _hip():
    """The runtime that this process has loaded."""
    for line in open("/proc/self/maps"):
        path = line.split()[-1]
        if "libamdhip64.so" in path:
            return ctypes.CDLL(path)
    raise RuntimeError("no HIP runtime is loaded")


def count(call):
    """call(stream) makes the launches on that stream, and has been made once before."""
    import torch
    bx.lib()
    torch.cuda.synchronize()
    hip, stream = _hip(), torch.cuda.Stream()
    s, graph, n = ctypes.c_void_p(stream.cuda_stream), ctypes.c_void_p(), ctypes.c_size_t()
    assert hip.hipStreamBeginCapture(s, 2) == 0                 # relaxed
    try:
        call(stream)
    finally:
        assert hip.hipStreamEndCapture(s, ctypes.byref(graph)) == 0
    assert hip.hipGraphGetNodes(graph, None, ctypes.byref(n)) == 0
    assert hip.hipGraphDestroy(graph) == 0
    return n.value
