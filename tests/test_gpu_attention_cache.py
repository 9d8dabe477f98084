"""Attention of one or a few queries per sequence over the int8 cache, against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_kv_cache import IDS, TYPES, cache_of, gen, ints, rows_at, table_of  # noqa: E402


def definition(q, cache, table, lengths, page, scale=None):
    """(out, how far the kernel's may be from it). q [batch, queries, heads, d].

    Roundings. q as fp16 of its row's power of two: exact, or off by half of fp16's smallest number, 2^-25, times
    at most twice the row's largest: d 2^-24 max|q| max|k| in a score. A score's sum over d products in fp32, cut off at
    each step: (d + 8) 2^-23 sum |q||k|. Its two factors and the difference from the maximum: 4 2^-24 (|t| + |t - m|), with
    |m| <= max |t|, and 2^-22 for the power: all times 2 for sum and total. A probability as fp16: 2^-11, or 2^-25 of
    2^-6, of V's largest scale: n 2^-30 max |v| in all. Sums over blocks, cut off, warps and parts: (n / 16 + 400) 2^-23.
    The result: half a step of its type."""
    batch, n, heads, d = q.shape
    kv = cache.k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    off = torch.zeros_like(out)
    eps = torch.finfo(q.dtype).eps
    for b in range(batch):
        length = int(lengths[b])
        if length <= 0:
            continue
        k, v = (x.double() for x in rows_at(cache, table, b, length, page, torch.float64))
        for i in range(n):
            m = length - n + 1 + i
            if m <= 0:
                continue
            for h in range(heads):
                x, keys, values = q[b, i, h].double(), k[:m, h * kv // heads], v[:m, h * kv // heads]
                t = keys @ x * scale
                p = torch.exp(t - t.max())
                size = (keys.abs() @ x.abs()).max() * abs(scale)
                error = (d + 8) * 2.0 ** -23 * size + d * 2.0 ** -24 * float(x.abs().max() * keys.abs().max()) * abs(scale)
                error += 12 * 2.0 ** -24 * float(t.abs().max()) + 2.0 ** -22
                relative = 2.0 ** -11 + 2 * math.expm1(min(50.0, float(error))) + (m / 16 + 400) * 2.0 ** -23
                out[b, i, h] = p @ values / p.sum()
                off[b, i, h] = (p @ values.abs() / p.sum()) * relative + m * 2.0 ** -30 * values.abs().max()
    off += out.abs() * eps / 2 + torch.finfo(q.dtype).tiny * eps
    return out, off * 1.001


def check(got, q, cache, table, lengths, page, scale=None):
    wide = q if q.dim() == 4 else q[:, None]
    want, off = definition(wide, cache, table, lengths, page, scale)
    far = (got.double().view(wide.shape) - want).abs() / off
    assert got.dtype == q.dtype and got.shape == q.shape
    assert bool((far <= 1).all()), float(far.max())


CASES = [  # lengths, queries, heads, kv, d, page
    ([1], 1, 1, 1, 16, 16), ([2], 1, 8, 1, 128, 16), ([15], 1, 4, 4, 64, 16), ([16], 1, 8, 2, 128, 64),
    ([17], 1, 7, 7, 32, 32), ([127, 128, 129], 1, 16, 2, 128, 16), ([2047], 1, 32, 8, 128, 64),
    ([0, 5, 0, 300], 1, 10, 2, 80, 48), ([1000, 1, 33, 4097], 1, 9, 1, 96, 128), ([700, 31], 1, 40, 2, 112, 64),
    ([600, 77], 1, 33, 1, 48, 16), ([300], 2, 4, 4, 64, 16), ([3, 50, 0, 2, 1], 4, 8, 2, 128, 16),
    ([1, 40], 7, 6, 2, 64, 32), ([130], 33, 4, 2, 128, 16), ([5], 16, 5, 1, 64, 16), ([9000], 1, 2, 1, 64, 256),
    ([20 + 13 * i for i in range(70)], 1, 4, 2, 64, 16), ([40000], 1, 8, 1, 128, 64),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lengths,queries,heads,kv,d,page", CASES, ids=range(len(CASES)))
def test_attention(lengths, queries, heads, kv, d, page, dtype):
    table, pages = table_of(lengths, page, 1)
    cache = cache_of(pages, kv, page, d, 2)
    shape = (len(lengths), heads, d) if queries == 1 else (len(lengths), queries, heads, d)
    q = torch.randn(shape, generator=gen(3), device="cuda").to(dtype)
    got = ops.attention_cache_s8(q, cache, table, ints(lengths))
    check(got, q, cache, table, lengths, page)
    assert ops.device_status() == 0
    again = ops.attention_cache_s8(q, cache, table, ints(lengths))
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_scales_of_scores(scale, dtype):
    """Scores from all alike to ones that leave a single position, either sign."""
    table, pages = table_of([333], 16, 1)
    cache = cache_of(pages, 2, 16, 64, 2)
    q = torch.randn((1, 6, 64), generator=gen(3), device="cuda").to(dtype)
    check(ops.attention_cache_s8(q, cache, table, ints([333]), scale=scale), q, cache, table, [333], 16, scale)


def test_magnitudes():
    """Rows of queries from the smallest to the largest, scales of blocks far apart, a maximum that rises to the end."""
    table, pages = table_of([800], 16, 1)
    cache = cache_of(pages, 1, 16, 64, 2)
    powers = torch.randint(-12, 8, cache.v_scales.shape, generator=gen(5), device="cuda")
    cache.v_scales.mul_(torch.ldexp(torch.ones_like(cache.v_scales), powers))
    order = table[0, :50].long()
    cache.k_scales[order, 0, 0] *= torch.linspace(0.01, 6, 50, device="cuda")
    q = torch.randn((1, 8, 64), generator=gen(3), device="cuda").bfloat16()
    q[0, :, 0] = 3
    q *= torch.tensor([2.0 ** e for e in (-126, -60, -20, -3, 0, 1, 2, 3)], device="cuda").bfloat16()[:, None]
    check(ops.attention_cache_s8(q, cache, table, ints([800])), q, cache, table, [800], 16)
    cache.v_scales.mul_(2.0 ** -60)
    check(ops.attention_cache_s8(q, cache, table, ints([800])), q, cache, table, [800], 16)


def test_bad_values_stay_with_the_queries_that_see_them():
    table, pages = table_of([64, 64], 16, 1)
    cache = cache_of(pages, 2, 16, 64, 2)
    q = torch.randn((2, 3, 4, 64), generator=gen(3), device="cuda").bfloat16()
    lengths = ints([50, 50])
    want = ops.attention_cache_s8(q, cache, table, lengths)
    # blocks behind the last position, other heads, other sequences
    cache.k_scales[table[0, 3].long(), 0, 0] = float("nan")  # positions 48 .., of which queries 1 and 2 see some
    cache.v_scales[table[1, 0].long(), 1, 0] = float("inf")
    cache.v_scales[table[1, 3].long(), 0, 0] = float("inf")
    got = ops.attention_cache_s8(q, cache, table, lengths)
    same = torch.ones((2, 3, 4), dtype=torch.bool, device="cuda")
    same[0, 1:, :2] = False
    same[1, :, 2:] = False
    same[1, 1:, :2] = False
    assert torch.equal(got[same], want[same])
    assert bool(torch.isnan(got[0, 1:, :2]).all())
    assert not bool(torch.isfinite(got[~same]).any())
    assert bool((ops.attention_cache_s8(q, cache, table, ints([48, 0]))[1] == 0).all())
    assert bool(torch.isfinite(ops.attention_cache_s8(q, cache, table, ints([48, 0]))).all())


def test_queries_with_nan_and_infinity():
    table, pages = table_of([40], 16, 1)
    cache = cache_of(pages, 1, 16, 64, 2)
    q = torch.randn((1, 4, 64), generator=gen(3), device="cuda").bfloat16()
    want = ops.attention_cache_s8(q, cache, table, ints([40]))
    q[0, 1, 3], q[0, 2, 60] = float("nan"), float("inf")
    got = ops.attention_cache_s8(q, cache, table, ints([40]))
    assert torch.equal(got[0, ::3], want[0, ::3]) and bool(torch.isnan(got[0, 1:3]).all())


def test_strides_alignment_and_results_of_the_caller():
    table, pages = table_of([90, 200], 16, 1)
    cache = cache_of(pages, 2, 16, 64, 2)
    flat = torch.randn((2, 3, 500), generator=gen(3), device="cuda").half()
    q = flat[:, :, 3:3 + 4 * 67].unflatten(2, (4, 67))[..., :64]
    out = torch.full((6, 5, 80), 7.0, device="cuda").half()
    part = out.view(2, 3, 5, 80)[:, :, :4, 1:65]
    got = ops.attention_cache_s8(q, cache, table, ints([90, 200]), out=part)
    assert got.data_ptr() == part.data_ptr()
    assert torch.equal(part, ops.attention_cache_s8(q.contiguous(), cache, table, ints([90, 200])))
    rest = out.clone()
    rest.view(2, 3, 5, 80)[:, :, :4, 1:65] = 7
    assert bool((rest == 7).all())


def test_pages_that_are_not_there_are_not_seen():
    table, pages = table_of([64], 16, 1)
    cache = cache_of(pages, 1, 16, 64, 2)
    q = torch.randn((1, 4, 64), generator=gen(3), device="cuda").half()
    holes = table.clone()
    holes[0, 1], holes[0, 2] = -1, pages
    got = ops.attention_cache_s8(q, cache, holes, ints([64]))
    torch.cuda.synchronize()
    assert ops.device_status() == 0x201
    short = torch.stack([table[0, 0], table[0, 3]])[None].contiguous()
    assert bool(torch.isfinite(got).all())
    check(got, q, cache, short, [32], 16)
    got = ops.attention_cache_s8(q, cache, table[:, :4].contiguous(), ints([10 ** 9]))  # longer than the table
    torch.cuda.synchronize()
    assert ops.device_status() == 0x201
    check(got, q, cache, table, [64], 16)


def test_calls_at_the_same_time():
    """Two streams, each with workspaces of its own, and what a call waits for on its own stream."""
    table, pages = table_of([3000, 100], 16, 1)
    cache = cache_of(pages, 2, 16, 64, 2)
    qs = [torch.randn((2, 8, 64), generator=gen(s), device="cuda").half() for s in range(2)]
    want = [ops.attention_cache_s8(q, cache, table, ints([3000, 100])) for q in qs]
    lengths = ints([3000, 100])
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for s, q, g in zip(streams, qs, got):
            with torch.cuda.stream(s):
                g.append(ops.attention_cache_s8(q, cache, table, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_a_cache_of_more_than_two_to_the_31_bytes():
    """Pages from both ends of it."""
    pages, page = (1 << 31) // (8 * 128 * 128) + 9, 128
    cache = ops.kv_cache_s8(pages, 8, page, 128)
    small = cache_of(4, 8, page, 128, 2)
    where = torch.tensor([0, pages // 2, pages - 2, pages - 1], device="cuda")
    for big, part in zip(cache, small):
        big[where] = part
    table, near = where.int()[None].flip(1).contiguous(), ints([[3, 2, 1, 0]])
    q = torch.randn((1, 16, 128), generator=gen(3), device="cuda").bfloat16()
    got = ops.attention_cache_s8(q, cache, table, ints([500]))
    assert torch.equal(got, ops.attention_cache_s8(q, small, near, ints([500])))
    kr, vr = ops.kv_read_s8(cache, table, None, ints([0, 500]), 500)
    assert all(torch.equal(a, b) for a, b in zip((kr, vr), ops.kv_read_s8(small, near, None, ints([0, 500]), 500)))
    x = torch.randn((12, 8, 128), generator=gen(4), device="cuda").bfloat16()
    for c, t in ((cache, table), (small, near)):
        ops.kv_append_s8(c, t, ints([500]), x, x, cu_tokens=ints([0, 12]))
    assert all(torch.equal(big[where], part) for big, part in zip(cache, small))
