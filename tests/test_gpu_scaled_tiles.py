"""int8 products with scales per row and per output channel: few rows that go to the tensor-core tiles, tiles whose rows
lie apart, calls from several threads. Labelled calls are checked for the kernel that they take."""
import ctypes
import re
import threading

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


# Few rows of wide layers: boxes of 8 to 72 rows of activations, whose tiles' other rows are whatever lies behind them in
# shared memory; K whole, and cut over two, four and eight CTAs; fewer tiles than SMs, and more.
FEW = [(1, 14336, 4096), (8, 12000, 2064), (17, 9000, 4096), (24, 14336, 4096), (32, 8192, 4096), (40, 4096, 4096),
       (61, 14336, 4096), (5, 20000, 2064), (33, 19200, 640), (9, 20008, 2064), (48, 2048, 4096), (56, 520, 4112),
       (20, 8320, 8192), (65, 640, 8208)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", FEW)
def test_few_rows_by_tiles(m, n, k, dtype):
    a, b, sa, sb = whole((m, k), 1), whole((n, k), 2), scales(m, 3), scales(n, 4)
    bias = torch.randn((n,), generator=gen(6), device="cuda") if m % 2 else None
    check_product(ops.matmul_s8_scaled(a, b, sa, sb, bias, dtype), a, sa, b, sb, bias)
    names = kernels_of(lambda: ops.matmul_s8_scaled(a, b, sa, sb, bias, dtype))
    assert set(names) == {"product_split"}


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


# Rows of an odd length in whole units, of both operands: what stands behind a row in its last unit counts for nothing,
# in tiles and where little of everything is streamed.
@pytest.mark.parametrize("m,k,pitch,by", [(20000, 1001, 1008, "tiles"), (9000, 127, 128, "stream"),
                                          (20000, 17, 32, "tiles")])
def test_odd_rows_in_whole_units(m, k, pitch, by):
    buf, wbuf = torch.full((m, pitch), 77, dtype=torch.int8, device="cuda"), torch.full((2048,), 55, dtype=torch.int8,
                                                                                       device="cuda")
    a, b = buf[:, :k], wbuf[:k].view(1, k)
    a.copy_(whole((m, k), 1))
    b.copy_(whole((1, k), 2))
    sa, sb = scales(m, 3), scales(1, 4)
    check_product(ops.matmul_s8_scaled(a, b, sa, sb), a, sa, b, sb, None)
    names = kernels_of(lambda: ops.matmul_s8_scaled(a, b, sa, sb))
    assert len(names) == 1 and (names[0] == "product_stream") == (by == "stream")
    x = torch.full((m, pitch), 1e30, device="cuda")[:, :k]
    x.copy_(torch.randn((m, k), generator=gen(5), device="cuda"))
    q, sx = rows_of(x)
    check_product(ops.linear_s8(x, b, sb), q, sx, b, sb, None)


# Threads with a stream each, at once: results are those of one call alone, and no thread ends early.
def test_threads_at_once_all_finish():
    b, sb = whole((4096, 1040), 2), scales(4096, 4)
    xs = [torch.randn((m, 1040), generator=gen(m), device="cuda").half() for m in (1, 20, 100, 700)]
    wants = [ops.linear_s8(x, b, sb) for x in xs]
    torch.cuda.synchronize()
    turns, finished, failed = 25, [], []

    def work(order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in order * turns:
                    if not torch.equal(ops.linear_s8(xs[i], b, sb), wants[i]):
                        failed.append(f"{xs[i].shape[0]} rows differ")
            finished.append(order)
        except BaseException as e:  # (a thread's exception ends nothing but the thread)
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(order,)) for order in ([0, 1, 2, 3], [3, 1, 0, 2], [2, 3, 1, 0])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and len(finished) == len(threads)
