"""What the int8 operators with run-time scales refuse, before anything is launched (no GPU needed)."""
import pytest
import torch

from megcc_b200 import _lib, ops

NULL_PTR, OUT_OF_RANGE, DTYPE, LAYOUT = 1, 4, 11, 12
P = 4096  # an address that nothing reads


def quantize(x=P, dtype=0, m=2, k=64, ldx=64, q=P, ldq=64, scales=P):
    return _lib.lib().mb200_quantize_rows_s8(x, dtype, m, k, ldx, q, ldq, scales, None)


def product(m=2, n=8, k=64, a=P, lda=64, b=P, sa=P, sb=P, bias=None, c=P, dtype=0, ldc=8, ws=None, nbytes=0):
    return _lib.lib().mb200_matmul_s8_scaled(m, n, k, a, lda, b, sa, sb, bias, c, dtype, ldc, ws, nbytes, None)


def linear(m=2, n=8, k=64, x=P, dtype=0, ldx=64, b=P, sb=P, bias=None, y=P, ldy=8, ws=None, nbytes=0):
    return _lib.lib().mb200_linear_s8(m, n, k, x, dtype, ldx, b, sb, bias, y, ldy, ws, nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), NULL_PTR), (dict(q=None), NULL_PTR), (dict(scales=None), NULL_PTR),
    (dict(dtype=3), DTYPE), (dict(dtype=-1), DTYPE), (dict(m=-1), LAYOUT), (dict(k=0), LAYOUT),
    (dict(ldx=63), LAYOUT), (dict(ldq=10), LAYOUT), (dict(x=P + 2), LAYOUT), (dict(x=P + 1, dtype=1), LAYOUT),
    (dict(scales=P + 1), LAYOUT), (dict(m=0, x=None, q=None, scales=None), 0)])
def test_quantize_rows(change, status):
    assert quantize(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(a=None), NULL_PTR), (dict(b=None), NULL_PTR), (dict(sa=None), NULL_PTR), (dict(sb=None), NULL_PTR),
    (dict(c=None), NULL_PTR), (dict(dtype=7), DTYPE), (dict(m=-3), LAYOUT), (dict(n=0), LAYOUT),
    (dict(k=-1), LAYOUT), (dict(k=131072, lda=131072), OUT_OF_RANGE), (dict(lda=60), LAYOUT),
    (dict(ldc=7), LAYOUT), (dict(sa=P + 2), LAYOUT), (dict(sb=P + 2), LAYOUT), (dict(bias=P + 1), LAYOUT),
    (dict(c=P + 2), LAYOUT), (dict(c=P + 1, dtype=2), LAYOUT), (dict(m=0, a=None, b=None, c=None), 0),
    (dict(m=2 ** 31 - 511), OUT_OF_RANGE), (dict(n=2 ** 31 - 1, ldc=2 ** 31), OUT_OF_RANGE)])
def test_product(change, status):
    assert product(**change) == status
    if status:
        assert b"matmul_s8_scaled" in _lib.lib().mb200_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(x=None), NULL_PTR), (dict(b=None), NULL_PTR), (dict(sb=None), NULL_PTR), (dict(y=None), NULL_PTR),
    (dict(dtype=3), DTYPE), (dict(m=-3), LAYOUT), (dict(n=0), LAYOUT), (dict(k=0), LAYOUT),
    (dict(k=200000, ldx=200000), OUT_OF_RANGE), (dict(ldx=60), LAYOUT), (dict(ldy=7), LAYOUT),
    (dict(x=P + 2), LAYOUT), (dict(sb=P + 2), LAYOUT), (dict(bias=P + 1), LAYOUT),
    (dict(y=P + 1, dtype=1), LAYOUT), (dict(m=0, x=None), 0), (dict(m=2 ** 31 - 1), OUT_OF_RANGE),
    (dict(n=2 ** 31 - 511, ldy=2 ** 31), OUT_OF_RANGE)])
def test_linear(change, status):
    assert linear(**change) == status


def test_python_calls_want_matrices_on_the_gpu():
    x, b, s = torch.zeros(2, 64), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for call in (lambda: ops.quantize_rows_s8(x), lambda: ops.linear_s8(x, b, s),
                 lambda: ops.matmul_s8_scaled(b, b, s, s), lambda: ops.linear_s8(x.double(), b, s)):
        with pytest.raises(ValueError):
            call()


def moe(tokens=2, d=64, f=32, experts=4, top_k=2, renormalize=1, dtype=2, x=P, ldx=64, logits=P, w1=P, s1=P, w2=P,
        s2=P, y=P, ldy=64, ws=P, nbytes=1 << 30):
    import ctypes
    p = _lib.MoeParam(tokens, d, f, experts, top_k, renormalize, dtype)
    return _lib.lib().mb200_moe_s8(ctypes.byref(p), x, ldx, logits, w1, s1, w2, s2, y, ldy, ws, nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), NULL_PTR), (dict(logits=None), NULL_PTR), (dict(w1=None), NULL_PTR), (dict(s1=None), NULL_PTR),
    (dict(w2=None), NULL_PTR), (dict(s2=None), NULL_PTR), (dict(y=None), NULL_PTR), (dict(ws=None), NULL_PTR),
    (dict(dtype=3), DTYPE), (dict(tokens=-1), LAYOUT), (dict(d=0), LAYOUT), (dict(f=0), LAYOUT),
    (dict(experts=0), LAYOUT), (dict(top_k=0), LAYOUT), (dict(top_k=5), LAYOUT), (dict(tokens=65), OUT_OF_RANGE),
    (dict(experts=513), OUT_OF_RANGE), (dict(experts=40, top_k=17), OUT_OF_RANGE),
    (dict(d=16385, ldx=30000, ldy=30000), OUT_OF_RANGE), (dict(tokens=9, d=8193, ldx=30000, ldy=30000), OUT_OF_RANGE),
    (dict(f=131072), OUT_OF_RANGE), (dict(ldx=63), LAYOUT), (dict(ldy=63), LAYOUT), (dict(x=P + 1), LAYOUT),
    (dict(y=P + 1), LAYOUT), (dict(logits=P + 2), LAYOUT), (dict(s1=P + 2), LAYOUT), (dict(s2=P + 1), LAYOUT),
    (dict(ws=P + 128), LAYOUT), (dict(nbytes=100), LAYOUT), (dict(tokens=0, x=None, ws=None), 0)])
def test_moe(change, status):
    assert moe(**change) == status


def test_moe_workspace_and_null_parameters():
    import ctypes
    size = _lib.lib().mb200_moe_s8_workspace_bytes
    assert size(None) == 0 and _lib.lib().mb200_moe_s8(None, *[P, 64] + [P] * 6 + [64, P, 0, None]) == NULL_PTR
    p = _lib.MoeParam(2, 64, 33, 4, 2, 1, 2)
    assert size(ctypes.byref(p)) == 256 + 256 + 256  # 4 slots of 64 whole numbers, of 2 scales, the routing
    p.tokens = 65
    assert size(ctypes.byref(p)) == 0
