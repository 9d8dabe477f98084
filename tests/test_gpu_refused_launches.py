"""A launch that the runtime refuses is reported by the call that made it, once: the calls behind it, of this library or
another one, find no error of it."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import _lib, ops  # noqa: E402

RUNTIME = 3


@pytest.fixture
def legacy_stream_refused():
    """While a blocking stream captures, the runtime refuses every launch on the legacy default stream."""
    rt = ctypes.CDLL("libcudart.so.12")
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.cudaStreamCreate(ctypes.byref(stream)) == 0
    torch.cuda.synchronize()

    def begin():
        assert rt.cudaStreamBeginCapture(stream, 1) == 0  # (of this thread)

    def end():
        rt.cudaStreamEndCapture(stream, ctypes.byref(graph))
        rt.cudaGetLastError()

    yield begin, end, rt.cudaPeekAtLastError
    rt.cudaStreamDestroy(stream)
    rt.cudaGetLastError()


def calls():
    lib, p = _lib.lib(), ctypes.c_void_p
    x = torch.randn((300, 528), device="cuda")
    q = torch.ones((300, 528), dtype=torch.int8, device="cuda")
    b = torch.ones((512, 528), dtype=torch.int8, device="cuda")
    s, y = torch.ones(512, device="cuda"), torch.zeros((300, 528), device="cuda")
    ws = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    logits, w1 = torch.zeros((64, 4), device="cuda"), torch.ones((4, 64, 64), dtype=torch.int8, device="cuda")
    keep = (x, q, b, s, y, ws, logits, w1)

    def product(m, k, a=q, n=512):
        return lambda: lib.mb200_matmul_s8_scaled(m, n, k, p(a.data_ptr()), k, p(b.data_ptr()), p(s.data_ptr()),
                                                  p(s.data_ptr()), None, p(y.data_ptr()), 0, 512, p(ws.data_ptr()),
                                                  ws.numel(), None)

    def linear(m):
        return lambda: lib.mb200_linear_s8(m, 512, 528, p(x.data_ptr()), 0, 528, p(b.data_ptr()), p(s.data_ptr()), None,
                                           p(y.data_ptr()), 512, p(ws.data_ptr()), ws.numel(), None)

    def moe(t):
        param = _lib.MoeParam(t, 64, 32, 4, 2, 1, 0)
        return lambda: lib.mb200_moe_s8(ctypes.byref(param), p(x.data_ptr()), 64, p(logits.data_ptr()),
                                        p(w1.data_ptr()), p(s.data_ptr()), p(b.data_ptr()), p(s.data_ptr()),
                                        p(y.data_ptr()), 64, p(ws.data_ptr()), ws.numel(), None)

    return keep, {
        "quantize": lambda: lib.mb200_quantize_rows_s8(p(x.data_ptr()), 0, 300, 528, 528, p(q.data_ptr()), 528,
                                                       p(y.data_ptr()), None),
        "stream": product(4, 528), "tiles": product(300, 528), "pad": product(256, 523),
        "linear": linear(2), "linear_rows": linear(300), "moe_few": moe(2), "moe": moe(20)}


def test_refused_launches_leave_no_error(legacy_stream_refused):
    begin, end, left_behind = legacy_stream_refused
    keep, by_name = calls()
    for name, call in by_name.items():
        assert call() == 0, (name, _lib.lib().mb200_last_error())
    torch.cuda.synchronize()
    for name, call in by_name.items():
        begin()
        status, left = call(), left_behind()
        end()
        assert status == RUNTIME, name
        assert left == 0, name
        assert call() == 0, (name, _lib.lib().mb200_last_error())
    torch.cuda.synchronize()
    assert ops.linear_s8(keep[0], keep[2], keep[3]).shape == (300, 512)
