"""int8 operators with run-time scales past 2^31 elements of each operand, and in the smallest layers; results whose rows
lie apart in tiles with K cut; workspaces of any content."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from megcc_b200._lib import check as ok, lib  # noqa: E402
from test_gpu_moe import check as check_moe, layer  # noqa: E402
from test_gpu_scaled import IDS, TYPES, check_product, gen, rows_of, scales, whole  # noqa: E402


def ends(n):
    """A few rows from both ends of n, and from the middle."""
    return sorted({0, 1, n // 2, n - 130, n - 2, n - 1} & set(range(n)))


def check_rows(got, q, sa, b, sb, rows):
    check_product(got[rows], q, sa, b, sb, None)


# results of 2.8e9 elements, stored by the TMA and by warps (whose columns are odd)
@pytest.mark.parametrize("n", [40000, 40001])
def test_results_past_32_bits(n):
    m, k = 70000, 64
    a, b, sa, sb = whole((m, k), 1), whole((n, k), 2), scales(m, 3), scales(n, 4)
    got = ops.matmul_s8_scaled(a, b, sa, sb, None, torch.float16)
    rows = ends(m)
    check_rows(got, a[rows], sa[rows], b, sb, rows)


# activations of 2.8e9 elements, through their whole numbers
@pytest.mark.parametrize("k", [40000, 39999])
def test_activations_past_32_bits(k):
    m, n = 70000, 64
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda").normal_(generator=gen(1))
    b, sb = whole((n, k), 2), scales(n, 4)
    rows = ends(m)
    q, sa = rows_of(x[rows])
    check_rows(ops.linear_s8(x, b, sb), q, sa, b, sb, rows)


# weights of 2.4e9 elements: streamed, by tiles, and laid out anew
@pytest.mark.parametrize("m,k", [(1, 40000), (9, 40000), (40, 40000), (1, 39999), (40, 39999)])
def test_weights_past_32_bits(m, k):
    n = 60000
    b, sb = whole((n, k), 2), scales(n, 4)
    a, sa = whole((m, k), 1), scales(m, 3)
    got = ops.matmul_s8_scaled(a, b, sa, sb)
    cols = ends(n)
    check_product(got[:, cols], a, sa, b[cols], sb[cols], None)


def test_rows_far_apart():
    m, k, pitch = 3, 96, (1 << 31) + 16
    buf = torch.empty((2 * pitch + k,), dtype=torch.int8, device="cuda")
    a = buf.as_strided((m, k), (pitch, 1))
    a.copy_(whole((m, k), 1))
    b, sa, sb = whole((40, k), 2), scales(m, 3), scales(40, 4)
    check_product(ops.matmul_s8_scaled(a, b, sa, sb), a, sa, b, sb, None)


# experts whose weights pass 2^31 bytes, the last of them chosen
@pytest.mark.parametrize("t", [2, 20])
def test_experts_past_32_bits(t):
    x, _, _, s1, _, s2 = layer(t, 4096, 1024, 2, 3)
    e = 512
    w1 = torch.empty((e, 2048, 4096), dtype=torch.int8, device="cuda").random_(-128, 128, generator=gen(5))
    w2 = torch.empty((e, 4096, 1024), dtype=torch.int8, device="cuda").random_(-128, 128, generator=gen(6))
    s1, s2 = s1[:1].expand(e, -1).contiguous(), s2[:1].expand(e, -1).contiguous()
    logits = torch.randn((t, e), generator=gen(7), device="cuda")
    logits[:, 505:] += 6
    check_moe((x, logits, w1, s1, w2, s2), 3, True)


@pytest.mark.parametrize("t,d,f,e,top", [(1, 1, 1, 1, 1), (5, 1, 1, 3, 2), (9, 3, 2, 7, 7), (64, 2, 33, 2, 2),
                                         (3, 15, 1, 16, 16)])
def test_the_smallest_experts(t, d, f, e, top):
    check_moe(layer(t, d, f, e, t + d, torch.float32), top, True)


def call(m, n, k, x, b, sb, y, ldy, fill, sa=None):
    """linear_s8, or matmul_s8_scaled with the rows' scales, in a workspace full of `fill`."""
    kind = TYPES.index(y.dtype)
    if sa is None:
        nbytes = lib().mb200_linear_s8_workspace_bytes(m, n, k, b.data_ptr())
    else:
        nbytes = lib().mb200_matmul_s8_scaled_workspace_bytes(m, n, k, x.data_ptr(), x.stride(0), b.data_ptr())
    ws = torch.full((nbytes + 512,), fill, dtype=torch.uint8, device="cuda")
    base = ws.data_ptr() + -ws.data_ptr() % 256
    p = ctypes.c_void_p
    if sa is None:
        ok(lib().mb200_linear_s8(m, n, k, p(x.data_ptr()), kind, x.stride(0), p(b.data_ptr()), p(sb.data_ptr()), None,
                                 p(y.data_ptr()), ldy, p(base), nbytes, ops._stream()))
    else:
        ok(lib().mb200_matmul_s8_scaled(m, n, k, p(x.data_ptr()), x.stride(0), p(b.data_ptr()), p(sa.data_ptr()),
                                        p(sb.data_ptr()), None, p(y.data_ptr()), kind, ldy, p(base), nbytes,
                                        ops._stream()))
    end = base - ws.data_ptr() + nbytes
    assert bool((ws[end:] == fill).all()) and bool((ws[:base - ws.data_ptr()] == fill).all())


# Tiles with K whole and cut over two, four and eight CTAs, results at any element and rows apart; the workspace holds
# anything, and nothing else is written.
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k,offset,pitch", [(61, 14337, 2048, 3, 14341), (130, 4200, 1601, 0, 4208),
                                                (128, 2002, 4096, 8, 2008), (100, 201, 6400, 1, 203),
                                                (56, 518, 4112, 0, 520), (300, 902, 201, 4, 904),
                                                (24, 2100, 4097, 0, 2104), (9, 4100, 2049, 5, 4101)])
def test_tiles_of_rows_apart_in_any_workspace(m, n, k, offset, pitch, dtype):
    x = torch.randn((m, k), generator=gen(1), device="cuda").to(dtype)
    a, sa = whole((m, k), 5), scales(m, 3)
    b, sb = whole((n, k), 2), scales(n, 4)
    q, sx = rows_of(x)
    for fill in (0, 255, 127):
        for rows, scale, given in ((q, sx, None), (a, sa, sa)):
            buf = torch.full((offset + (m + 3) * pitch + 300,), 7.0, device="cuda", dtype=dtype)
            y = buf.as_strided((m, n), (pitch, 1), offset)
            call(m, n, k, x if given is None else a, b, sb, y, pitch, fill, given)
            check_product(y, rows, scale, b, sb, None)
            y.fill_(7.0)
            assert bool((buf == 7.0).all())
