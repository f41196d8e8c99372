"""Which kernels a call launches: their names and grids, from a captured graph of
it (hipGraphKernelNodeGetParams; nothing is replayed)."""
from __future__ import annotations

import ctypes as C
import re


class _Dim3(C.Structure):
    _fields_ = [("x", C.c_uint32), ("y", C.c_uint32), ("z", C.c_uint32)]


class _KernelNode(C.Structure):
    """hipKernelNodeParams (hip_runtime_api.h)."""
    _fields_ = [("block", _Dim3), ("extra", C.c_void_p), ("func", C.c_void_p), ("grid", _Dim3), ("params", C.c_void_p),
                ("shared", C.c_uint32)]


def _hip():
    for line in open("/proc/self/maps"):  # the runtime that torch has loaded
        if "libamdhip64.so" in line:
            return C.CDLL(line.split()[-1])
    raise RuntimeError("no HIP runtime is loaded")


def launches(call) -> dict[str, tuple[int, int, int]]:
    """kernel<its integer and boolean template arguments>: grid, of the kernels that
    call() launches, in order (each once).  call() has run before."""
    import torch
    hip = _hip()
    hip.hipKernelNameRefByPtr.restype = C.c_char_p
    hip.hipKernelNameRefByPtr.argtypes = [C.c_void_p, C.c_void_p]
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    graph, n = C.c_void_p(g.raw_cuda_graph()), C.c_size_t(0)
    assert hip.hipGraphGetNodes(graph, None, C.byref(n)) == 0
    nodes = (C.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(graph, nodes, C.byref(n)) == 0
    found = {}
    for node in nodes:
        p = _KernelNode()
        assert hip.hipGraphKernelNodeGetParams(C.c_void_p(node), C.byref(p)) == 0
        mangled = hip.hipKernelNameRefByPtr(p.func, None).decode()
        name = mangled[re.match(r"_ZN?(?:\d+_GLOBAL__N_1)?\d+", mangled).end():]
        m = re.match(r"(\w+?_kernel)(?:I((?:L[ib]\d+E)+)E)?", name)
        args = re.findall(r"L[ib](\d+)E", m.group(2) or "")
        found[f"{m.group(1)}<{', '.join(args)}>" if args else m.group(1)] = (p.grid.x, p.grid.y, p.grid.z)
    return found
