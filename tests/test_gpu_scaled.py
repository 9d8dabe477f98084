"""int8 products with scales per row and per output channel, against their definitions in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402

TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def whole(shape, seed):
    return torch.randint(-128, 128, shape, generator=gen(seed), device="cuda", dtype=torch.int8)


def scales(n, seed):
    return torch.rand((n,), generator=gen(seed), device="cuda") * 0.02 + 1e-3


def rows_of(x):
    """(whole numbers, scale) by definition: both factors are products of fp32 numbers with fp32 reciprocals (a
    quotient of fp32 numbers rounded to 64 and then to 32 bits is the correctly rounded one), x * inv is exact in
    64 bits."""
    x = x.double()
    amax = x.abs().amax(-1).clamp(min=2.0 ** -119)
    scale = (amax * float(torch.tensor(1 / 127, dtype=torch.float32))).float()
    inv = ((1 / amax).float().double() * 127).float().double()
    q = torch.round(x * inv[:, None])
    bad = ~torch.isfinite(x).all(-1)
    q[bad] = 0
    scale[bad] = float("nan")
    return q, scale


def product_bound(t, c, dtype):
    """Three roundings of the product's own terms (sum to fp32, two scales), one of the sum with the bias, one
    to the result's type (half a step, or half of the smallest number the type has)."""
    fi = torch.finfo(dtype)
    return (t.abs() * 3 * 2.0 ** -24 + c.abs() * (2.0 ** -24 + (fi.eps / 2 if dtype != torch.float32 else 0))) * 1.001 \
        + fi.tiny * fi.eps / 2


def check_product(got, q, sa, b, sb, bias):
    t = (q.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None]
    c = t if bias is None else t + bias.double()
    assert got.shape == c.shape
    off = (got.double() - c).abs()
    assert bool((off <= product_bound(t, c, got.dtype)).all()), float((off / product_bound(t, c, got.dtype)).max())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (3, 64), (1, 4096), (9, 129), (257, 512), (5, 1000),
                                 (4, 9001), (2, 40000), (1030, 96), (5, 20003), (2100, 4095)])
def test_quantize_rows(m, k, dtype):
    x = torch.randn((m, k), generator=gen(m + k), device="cuda").to(dtype)
    q, s = ops.quantize_rows_s8(x)
    want_q, want_s = rows_of(x)
    assert torch.equal(q.double(), want_q) and torch.equal(s, want_s)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_quantize_rows_of_special_values(dtype):
    x = torch.randn((11, 200), generator=gen(5), device="cuda")
    big = torch.finfo(dtype).max
    x = x.to(dtype)
    x[1] = 0
    x[2] = -0.0
    x[3, 17] = float("nan")
    x[4, 199] = float("inf")
    x[5, 0] = -float("inf")
    x[6] *= torch.finfo(dtype).tiny   # subnormals
    x[7] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    x[8, 3] = big
    x[9] = -big
    x[10] = torch.linspace(-1, 1, 200).to(dtype)  # halves of the largest: ties
    q, s = ops.quantize_rows_s8(x)
    want_q, want_s = rows_of(x)
    assert torch.equal(q.double(), want_q)
    assert torch.equal(s.nan_to_num(-1), want_s.nan_to_num(-1))
    assert s[3].isnan() and s[4].isnan() and s[5].isnan() and int(s.isnan().sum()) == 3


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("offset,pitch", [(0, 520), (1, 512), (3, 517), (8, 504), (0, 505)])
def test_quantize_rows_that_lie_apart(dtype, offset, pitch):
    buf = torch.randn((offset + 37 * pitch + 600,), generator=gen(pitch), device="cuda").to(dtype)
    x = buf.as_strided((37, 500), (pitch, 1), offset)
    q, s = ops.quantize_rows_s8(x)
    want_q, want_s = rows_of(x)
    assert torch.equal(q.double(), want_q) and torch.equal(s, want_s)


# Rows of numbers at any byte and any distance, what lies between them untouched
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,pitch,offset", [(3, 5, 7, 1), (7, 300, 303, 2), (1, 1, 1, 3), (2, 4097, 4097, 0),
                                              (2100, 2047, 2049, 1), (3, 9003, 9006, 3), (40, 256, 256, 5)])
def test_quantize_to_any_place(m, k, pitch, offset, dtype):
    from megcc_b200._lib import check, lib
    x = torch.randn((m, k), generator=gen(m + k), device="cuda").to(dtype)
    buf = torch.full((offset + m * pitch + 40,), 99, dtype=torch.int8, device="cuda")
    s = torch.empty(m, device="cuda")
    check(lib().mb200_quantize_rows_s8(x.data_ptr(), TYPES.index(dtype), m, k, k, buf.data_ptr() + offset, pitch,
                                       s.data_ptr(), ops._stream()))
    want_q, want_s = rows_of(x)
    q = buf.as_strided((m, k), (pitch, 1), offset)
    assert torch.equal(q.double(), want_q) and torch.equal(s, want_s)
    q.fill_(99)
    assert bool((buf == 99).all())


SIZES = [(1, 1, 1), (1, 16, 64), (1, 17, 63), (7, 1000, 512), (8, 130, 65), (9, 33, 4096), (16, 48, 48),
         (17, 100, 1000), (24, 1000, 512), (33, 257, 129), (64, 64, 2047), (65, 70, 272), (127, 300, 640),
         (128, 128, 128), (129, 129, 144), (200, 1000, 4099), (256, 512, 96), (300, 260, 16), (511, 136, 1040),
         (1000, 999, 333), (1, 5000, 11008), (2, 24, 131071), (1025, 2048, 256), (1, 100, 8000), (8, 64, 9000),
         # short sums of many columns; tiles of 192 and of 128 columns; K split over two, four and eight CTAs
         (2, 12735, 74), (7, 5000, 1024), (20, 9999, 130), (500, 9700, 1024), (256, 9472, 8192), (130, 4200, 1600),
         (128, 2000, 4096), (100, 200, 6400),
         # rows that no 16-byte copies take, of many weights
         (9, 4100, 2049), (24, 2100, 4097), (16, 9000, 1001), (148, 1614, 66), (300, 900, 201),
         # tiles of several turns, the last one partly filled
         (4001, 4000, 300), (3900, 3850, 208),
         # one row of tiles on more CTAs than SMs
         (70, 19072, 640), (3, 20000, 1280), (16, 40000, 1152)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul_s8_scaled(m, n, k, dtype):
    a, b, sa, sb = whole((m, k), 1), whole((n, k), 2), scales(m, 3), scales(n, 4)
    bias = torch.randn((n,), generator=gen(6), device="cuda") if (m + n) % 2 else None
    check_product(ops.matmul_s8_scaled(a, b, sa, sb, bias, dtype), a, sa, b, sb, bias)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_s8(m, n, k, dtype):
    x = (torch.randn((m, k), generator=gen(1), device="cuda") * 3).to(dtype)
    b, sb = whole((n, k), 2), scales(n, 4)
    bias = torch.randn((n,), generator=gen(6), device="cuda") if (m + n) % 2 else None
    q, sa = rows_of(x)
    got = ops.linear_s8(x, b, sb, bias)
    check_product(got, q, sa, b, sb, bias)
    # one call or two: the same bits
    q, sa = ops.quantize_rows_s8(x)
    assert torch.equal(got, ops.matmul_s8_scaled(q, b, sa, sb, bias, dtype))


# The longest sums of the largest products: -128 * -128 * 131071 still fits an int32.
@pytest.mark.parametrize("m", [1, 20, 200])
def test_sums_at_the_ends_of_an_int32(m):
    k = 131071
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((40, k), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    one = torch.ones(m, device="cuda")
    got = ops.matmul_s8_scaled(a, b, one, torch.ones(40, device="cuda"))
    want = a[:1].double() @ b.double().t()
    assert torch.equal(got, want.float().expand(m, 40))


# rows apart, bases and pitches at every alignment
@pytest.mark.parametrize("m", [5, 40, 150])
@pytest.mark.parametrize("offset,pitch", [(0, 528), (1, 512), (4, 516), (16, 513), (8, 520)])
def test_operands_anywhere(m, offset, pitch):
    buf = whole((offset + m * pitch + 600,), pitch)
    a = buf.as_strided((m, 512), (pitch, 1), offset)
    wbuf = whole((offset + 77 * 512 + 16,), 9)
    b = wbuf[offset:offset + 77 * 512].view(77, 512)
    sbuf = scales(m + 100, 4)
    sa, sb = sbuf[1:m + 1], sbuf[3:80]
    bias = torch.randn((80,), generator=gen(6), device="cuda")[1:78]
    check_product(ops.matmul_s8_scaled(a, b, sa, sb, bias), a, sa, b, sb, bias)
    x = torch.randn((offset + m * pitch + 600,), generator=gen(3), device="cuda").bfloat16()
    x = x.as_strided((m, 512), (pitch, 1), offset)
    q, sx = rows_of(x)
    check_product(ops.linear_s8(x, b, sb, bias), q, sx, b, sb, bias)


def call_linear(x, b, sb, y, ldy):
    from megcc_b200._lib import check, lib
    (m, k), n = x.shape, b.shape[0]
    nbytes = lib().mb200_linear_s8_workspace_bytes(m, n, k, b.data_ptr())
    ws = torch.empty(nbytes + 256, dtype=torch.uint8, device="cuda")
    base = ws.data_ptr() + -ws.data_ptr() % 256
    check(lib().mb200_linear_s8(m, n, k, x.data_ptr(), TYPES.index(x.dtype), x.stride(0), b.data_ptr(),
                                sb.data_ptr(), None, y.data_ptr(), ldy, base, nbytes, ops._stream()))


# What lies between and behind the rows of the result stays as it is.
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,offset,pitch", [(3, 33, 1, 40), (100, 136, 0, 144), (130, 120, 3, 121),
                                              (260, 264, 8, 272)])
def test_only_the_result_is_written(m, n, offset, pitch, dtype):
    x = torch.randn((m, 192), generator=gen(1), device="cuda").to(dtype)
    b, sb = whole((n, 192), 2), scales(n, 4)
    buf = torch.full((offset + (m + 3) * pitch + 300,), 7.0, device="cuda", dtype=dtype)
    y = buf.as_strided((m, n), (pitch, 1), offset)
    call_linear(x, b, sb, y, pitch)
    q, sa = rows_of(x)
    check_product(y, q, sa, b, sb, None)
    y.fill_(7.0)
    assert bool((buf == 7.0).all())


# A row without a scale (NaN, infinity) is NaN in the result, and no other row is.
@pytest.mark.parametrize("m", [2, 12, 140, 300])
def test_rows_without_a_scale(m):
    x = torch.randn((m, 320), generator=gen(1), device="cuda")
    x[0, 3] = float("inf")
    x[m - 1, 319] = float("nan")
    b, sb = whole((150, 320), 2), scales(150, 4)
    y = ops.linear_s8(x, b, sb)
    assert bool(y[0].isnan().all()) and bool(y[m - 1].isnan().all())
    q, sa = rows_of(x)
    if m > 2:
        check_product(y[1:m - 1], q[1:m - 1], sa[1:m - 1], b, sb, None)


@pytest.mark.parametrize("m", [1, 30, 200])
def test_no_rows_and_rows_of_zeros(m):
    b, sb = whole((100, 256), 2), scales(100, 4)
    bias = torch.randn((100,), generator=gen(6), device="cuda")
    assert ops.linear_s8(torch.empty((0, 256), device="cuda"), b, sb).shape == (0, 100)
    assert ops.matmul_s8_scaled(whole((0, 256), 1), b, scales(0, 1), sb).shape == (0, 100)
    assert ops.quantize_rows_s8(torch.empty((0, 256), device="cuda"))[0].shape == (0, 256)
    y = ops.linear_s8(torch.zeros((m, 256), device="cuda"), b, sb, bias)
    assert torch.equal(y, bias.expand(m, 100))


# The operands of one call may come from the call before it, weights among them, and a call may be captured
# and replayed, on another stream too.
@pytest.mark.parametrize("m", [1, 12, 100, 300])
def test_chains_streams_and_graphs(m):
    x = torch.randn((m, 512), generator=gen(1), device="cuda").half()
    w1t, w2 = whole((512, 768), 2), whole((256, 768), 3)
    s1, s2 = scales(768, 4) / 500, scales(256, 5)

    def chain(x):
        return ops.linear_s8(ops.linear_s8(x, ops.matmul_pack_b(w1t), s1), w2, s2)

    q, sa = rows_of(x)
    t = (q @ w1t.double()) * sa.double()[:, None] * s1.double()
    want = chain(x)
    # the first layer's result within its bound; the second against the definition on that very result
    h = ops.linear_s8(x, ops.matmul_pack_b(w1t), s1)
    assert bool(((h.double() - t).abs() <= product_bound(t, t, torch.float16)).all())
    q, sa = rows_of(h)
    check_product(want, q, sa, w2, s2, None)
    for _ in range(20):
        assert torch.equal(chain(x), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(x)
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            replayed = chain(x)
    side.synchronize()
    assert torch.equal(got, want)
    for seed in (7, 8):
        x.copy_(torch.randn((m, 512), generator=gen(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed, chain(x))


# A single row of either operand, or of the result, may name any pitch, whichever kernel takes it.
@pytest.mark.parametrize("m,n,k", [(1, 9600, 4096), (20000, 1, 1001), (20000, 1, 1008), (1, 1, 5), (9000, 1, 64)])
def test_single_rows(m, n, k):
    a, b, sa, sb = whole((m, k + 3), 1)[:, :k], whole((n, k), 2), scales(m, 3), scales(n, 4)
    check_product(ops.matmul_s8_scaled(a, b, sa, sb, None, torch.float16), a, sa, b, sb, None)
    x = torch.randn((m, k + 1), generator=gen(3), device="cuda").bfloat16()[:, :k]
    q, sx = rows_of(x)
    check_product(ops.linear_s8(x, b, sb), q, sx, b, sb, None)
    y = torch.zeros((m, n), device="cuda", dtype=x.dtype)
    call_linear(x, b, sb, y, n if m > 1 else 7)
    check_product(y, q, sx, b, sb, None)


# The longest row that an int counts: its last vector ends behind 2^31 elements.
def test_quantize_the_longest_row():
    k, part = 2 ** 31 - 1, 1 << 27
    x = torch.empty((1, k), dtype=torch.float16, device="cuda")
    for at in range(0, k, part):
        x[0, at:at + part].normal_(generator=gen(at + 1))
    x[0, k - 1] = 9.0
    q, s = ops.quantize_rows_s8(x)
    for at in range(0, k, part):
        piece = torch.cat([x[0, at:at + part], x[0, k - 1:]])[None]  # (the largest is the last)
        want_q, want_s = rows_of(piece)
        assert torch.equal(q[0, at:at + part].double(), want_q[0, :-1]) and torch.equal(s, want_s)


# A result that no GPU holds is torch's own error, and the next call works.
def test_results_larger_than_memory():
    b = torch.zeros((2 ** 21, 1), dtype=torch.int8, device="cuda")
    rows = torch.zeros((2 ** 21, 1), device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        ops.linear_s8(rows, b, torch.ones(2 ** 21, device="cuda"))
    assert ops.linear_s8(rows[:1], b, torch.ones(2 ** 21, device="cuda")).shape == (1, 2 ** 21)


# Two threads with a stream each, at once: results are those of one call alone.
def test_two_threads_at_once():
    import threading
    b, sb = whole((1000, 1040), 2), scales(1000, 4)
    xs = [torch.randn((m, 1040), generator=gen(m), device="cuda").half() for m in (1, 20, 100, 700)]
    wants = [ops.linear_s8(x, b, sb) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in order * 25:
                if not torch.equal(ops.linear_s8(xs[i], b, sb), wants[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(order,)) for order in ([0, 1, 2, 3], [3, 1, 0, 2])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# Kernels that do not overlap at all give the same bits.
def test_without_dependent_launches():
    from megcc_b200._lib import check, lib
    b, sb = whole((300, 519), 2), scales(300, 4)
    xs = [torch.randn((m, 519), generator=gen(m), device="cuda") for m in (1, 30, 400)]
    wants = [ops.linear_s8(x, b, sb) for x in xs]
    check(lib().mb200_set_option(b"pdl", 0))
    try:
        for x, want in zip(xs, wants):
            assert torch.equal(ops.linear_s8(x, b, sb), want)
    finally:
        check(lib().mb200_set_option(b"pdl", 1))


def test_addresses_past_32_bits():
    # 16400 rows of a pitch of 2^18 elements: the last ones lie more than 2^32 bytes in
    m, pitch = 16400, 1 << 18
    buf = torch.zeros((m * pitch,), dtype=torch.int8, device="cuda")
    a = buf.as_strided((m, 64), (pitch, 1))
    a.copy_(whole((m, 64), 1))
    b, sa, sb = whole((24, 64), 2), scales(m, 3), scales(24, 4)
    check_product(ops.matmul_s8_scaled(a, b, sa, sb), a, sa, b, sb, None)
