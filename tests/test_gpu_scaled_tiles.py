"""int8 products with scales per row and per output channel: tiles of the tensor cores whose rows of results
lie apart. Each call is checked for the kernel that it takes."""
import ctypes
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_scaled import IDS, TYPES, call_linear, check_product, gen, rows_of, scales, whole  # noqa: E402


class KernelNode(ctypes.Structure):
    """CUDA_KERNEL_NODE_PARAMS"""
    _fields_ = [("func", ctypes.c_void_p), ("sizes", ctypes.c_uint * 7), ("params", ctypes.c_void_p),
                ("extra", ctypes.c_void_p), ("kernel", ctypes.c_void_p), ("context", ctypes.c_void_p)]


def kernels_of(call):
    """Names of the kernels that a call launches, from the graph that captures it."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    driver = ctypes.CDLL("libcuda.so.1")
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert driver.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert driver.cuGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    names = []
    for node in nodes:
        p, name = KernelNode(), ctypes.c_char_p()
        assert driver.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
        if p.func:
            assert driver.cuFuncGetName(ctypes.byref(name), ctypes.c_void_p(p.func)) == 0
        else:
            assert driver.cuKernelGetName(ctypes.byref(name), ctypes.c_void_p(p.kernel)) == 0
        names.append(re.search(r"(\w+?)_kernel", re.sub(r"^.*?(?=product|quantize|pad)", "", name.value.decode()))[1])
    return names


# Rows of the result apart, by the TMA (rows of whole 16-byte units) and by warps, in tiles of 256 and 192 columns; what
# lies between and behind the rows stays as it is, within a row's last unit too.
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k,offset,pitch", [(2304, 2048, 512, 0, 2064), (600, 4896, 1040, 8, 4912),
                                                (1000, 19008, 256, 0, 19016), (2300, 2040, 512, 0, 2056),
                                                (600, 4890, 1040, 8, 4904), (600, 4896, 1040, 1, 4912),
                                                (600, 4890, 1040, 0, 4891)])
def test_wide_tiles_of_rows_apart(m, n, k, offset, pitch, dtype):
    x = torch.randn((m, k), generator=gen(1), device="cuda").to(dtype)
    b, sb = whole((n, k), 2), scales(n, 4)
    buf = torch.full((offset + (m + 3) * pitch + 300,), 7.0, device="cuda", dtype=dtype)
    y = buf.as_strided((m, n), (pitch, 1), offset)
    call_linear(x, b, sb, y, pitch)
    q, sa = rows_of(x)
    check_product(y, q, sa, b, sb, None)
    y.fill_(7.0)
    assert bool((buf == 7.0).all())
    names = kernels_of(lambda: ops.linear_s8(x, b, sb))
    assert names.count("product_pair") == 1 and names.count("product_split") == 0
