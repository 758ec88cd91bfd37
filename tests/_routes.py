"""Which kernels a call launches, by its captured graph."""

import ctypes
import re

import torch


def kernels_of(call, tmp_path):
    """The names of the kernels of one captured call, without `_kernel`; 256-row tiles that read 4-bit pages are `tiles_codes`."""
    call()  # (what is asked of a kernel once is asked outside the capture)
    graph, path = torch.cuda.CUDAGraph(keep_graph=True), tmp_path / "graph.dot"
    with torch.cuda.graph(graph):
        kept = call()
    assert ctypes.CDLL("libcuda.so.1").cuGraphDebugDotPrint(ctypes.c_void_p(graph.raw_cuda_graph()), str(path).encode(), 1) == 0
    del kept
    names = set()
    for name, codes in re.findall(r"_cu_[0-9a-f]{8}\d+([a-z][a-z0-9_]*?)_kernel(?:I\w*?Li\d+ELb([01])E)?", path.read_text()):
        names.add("tiles_codes" if name == "tiles" and codes == "1" else name)
    return names
