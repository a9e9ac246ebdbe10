"""Which kernels a call enqueues: the call is captured into a graph, which is not run, and its nodes are read. So a test that is
about one kernel can show that its sizes take that kernel, whatever the estimates behind the choice become."""
import ctypes

import torch

from util import load_package

pkg = load_package()


class _Dim3(ctypes.Structure):
    _fields_ = [("x", ctypes.c_uint), ("y", ctypes.c_uint), ("z", ctypes.c_uint)]


class _KernelNode(ctypes.Structure):
    _fields_ = [("block", _Dim3), ("extra", ctypes.c_void_p), ("func", ctypes.c_void_p), ("grid", _Dim3), ("params", ctypes.c_void_p), ("lds", ctypes.c_uint)]


def _check(rc):
    assert rc == 0, "hipError %d" % rc


def _demangled(name):
    name = name.replace(b"DF16b", b"u6__bf16")      # (older libraries take bf16's short form for something else)
    f = ctypes.CDLL("libstdc++.so.6").__cxa_demangle
    f.restype = ctypes.c_void_p
    status = ctypes.c_int()
    p = f(name, None, None, ctypes.byref(status))
    if status.value != 0:
        return name.decode()
    out = ctypes.string_at(p).decode()
    free = ctypes.CDLL(None).free
    free.argtypes = [ctypes.c_void_p]
    free(p)
    return out


def kernels_of(call):
    """Names (with template arguments) and grids of the kernels that call(stream) enqueues, in their order."""
    hip = pkg.lib()          # its own HIP runtime: symbols are looked up in what the library is linked to as well
    hip.hipKernelNameRefByPtr.restype = ctypes.c_char_p
    stream = torch.cuda.Stream()
    s = ctypes.c_void_p(int(stream.cuda_stream))
    graph, count = ctypes.c_void_p(), ctypes.c_size_t()
    torch.cuda.synchronize()
    _check(hip.hipStreamBeginCapture(s, ctypes.c_int(2)))        # relaxed: other threads' calls do not end it
    try:
        call(int(stream.cuda_stream))
    finally:
        _check(hip.hipStreamEndCapture(s, ctypes.byref(graph)))
    out = []
    _check(hip.hipGraphGetNodes(graph, None, ctypes.byref(count)))
    nodes = (ctypes.c_void_p * max(1, count.value))()
    _check(hip.hipGraphGetNodes(graph, nodes, ctypes.byref(count)))
    for node in nodes[:count.value]:
        kind, p = ctypes.c_int(), _KernelNode()
        _check(hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)))
        assert kind.value == 0, "a node that is no kernel"
        _check(hip.hipGraphKernelNodeGetParams(ctypes.c_void_p(node), ctypes.byref(p)))
        out.append((_demangled(hip.hipKernelNameRefByPtr(ctypes.c_void_p(p.func), None)), (p.grid.x, p.grid.y, p.grid.z)))
    _check(hip.hipGraphDestroy(graph))
    return out
