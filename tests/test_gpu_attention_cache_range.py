"""Attention over the int8 cache where its numbers lie far apart, with a bound of each row's own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_attention_cache import CASES  # noqa: E402
from test_gpu_kv_cache import IDS, TYPES, cache_of, gen, ints, rows_at, table_of  # noqa: E402


def row_bound(x, keys, values, weight, scale, dtype):
    """(out, how far the kernel's may be from it) of a query x over what it sees: keys and values [m, d] in 64 bits, weight
    [m] the scale of each position's values.

    Roundings. q as whole numbers of 22 bits of its row's power of two (of 2^-106 at least): off by half of one, 2^-21 of the
    row's largest. A score's products are exact, their sum is put together from two numbers in fp32, and multiplied by
    factors of five roundings: 2^-23 sum |q||k| + 8 2^-24 |t|. The difference from the maximum, of up to twice the
    largest score: 2^-23 max |t|; the power, 2^-22, and where the maximum rises or parts are joined others: 8 2^-22. All of it twice,
    for sum and total. p_j times its scale as fp16, 2^-11, or for fp16 results as two such numbers, 2^-21; or 2^-25 where 2^6 or
    more stands for the row's own largest p_j times scale, rounded up to a power of two: 2^-30 of that for each position and whole number.
    Sums, cut off: (m / 16 + 400) 2^-23. The result: half a step of its type."""
    d, m = keys.shape[1], keys.shape[0]
    t = keys @ x * scale
    p = torch.exp(t - t.max())
    p /= p.sum()
    size = float((keys.abs() @ x.abs()).max()) * abs(scale)
    grain = max(2.0 ** -21 * float(x.abs().max()), 2.0 ** -127) * float(keys.abs().sum(1).max()) * abs(scale)
    score = 2.0 ** -23 * size + grain + 10 * 2.0 ** -24 * float(t.abs().max()) + 8 * 2.0 ** -22
    held = 2.0 ** -21 if dtype == torch.float16 else 2.0 ** -11
    relative = held + 2 * math.expm1(min(50.0, score)) + (m / 16 + 400) * 2.0 ** -23
    out = p @ values
    off = (p @ values.abs()) * relative + m * 127 * 2.0 ** -30 * float((p * weight).max())
    off = off + out.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return out, off * 1.001


def check(got, q, cache, table, lengths, page, scale=None):
    """got, q: [batch, queries, heads, d]. The worst of each row's differences over its bound is at most 1."""
    batch, n, heads, d = q.shape
    kv = cache.k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    assert got.shape == q.shape and got.dtype == q.dtype
    most = 0.0
    for b in range(batch):
        capacity = table.shape[1] * page
        held = min(int(lengths[b]), capacity)
        if held <= 0:
            assert bool((got[b] == 0).all())
            continue
        k, v = (x.double() for x in rows_at(cache, table, b, held, page, torch.float64))
        where = torch.arange(held, device="cuda")
        weights = cache.v_scales[table[b, where // page].long(), :, where % page // 16].double()
        for i in range(n):
            m = min(int(lengths[b]) - n + 1 + i, held)
            for h in range(heads):
                g = h * kv // heads
                if m <= 0:
                    assert bool((got[b, i, h] == 0).all())
                    continue
                want, off = row_bound(q[b, i, h].double(), k[:m, g], v[:m, g], weights[:m, g], scale, q.dtype)
                most = max(most, float(((got[b, i, h].double() - want).abs() / off).max()))
    assert most <= 1, most


def against(cache, table, b, first, q, score, page=16):
    """Makes the block at position `first` of all heads one whose keys score about `score` with the first query of each group,
    and as much with the other sign for its opposite."""
    kv, d = cache.k.shape[1], cache.k.shape[3]
    number, o = int(table[b, first // page]), first % page
    for g in range(kv):
        x = q[g * (q.shape[0] // kv)].double()
        cache.k[number, g, o:o + 16] = (127 * x.sign()).to(torch.int8)
        cache.k_scales[number, g, o // 16] = score / (127 * float(x.abs().sum()) / math.sqrt(d))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("apart", [12, 24, 33, 40, 100])
@pytest.mark.parametrize("heads,kv,d,length,loud", [
    (4, 2, 64, 200, 0), (4, 2, 64, 200, 5), (4, 2, 128, 200, 12), (16, 1, 128, 200, 3), (12, 1, 80, 70, 2),
    (8, 1, 128, 5000, 0), (8, 1, 128, 5000, 200), (1, 1, 64, 129, 8)])
def test_a_loud_block_of_little_weight(heads, kv, d, length, loud, apart, dtype):
    """A block whose values are 2^apart times the others' and whose probability makes nothing of that."""
    table, pages = table_of([length], 16, 1)
    cache = cache_of(pages, kv, 16, d, 2)
    q = torch.randn((1, 1, heads, d), generator=gen(3), device="cuda").to(dtype)
    for g in range(kv):  # (queries of a group alike but for their size: the block is nothing to all of them)
        first = g * (heads // kv)
        q[0, 0, first:first + heads // kv] = q[0, 0, first] * torch.linspace(1, 1.5, heads // kv, device="cuda").to(dtype)[:, None]
    down = 2.0 ** (-90 if apart == 100 and dtype == torch.bfloat16 else -8)
    cache.v_scales.mul_(down)
    cache.v_scales[table[0, loud].long()] = 0.01 * down * 2.0 ** apart
    against(cache, table, 0, loud * 16, q[0, 0], -(apart + 22) * math.log(2))
    got = ops.attention_cache_s8(q[:, 0].contiguous(), cache, table, ints([length]))
    check(got[:, None], q, cache, table, [length], 16)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("apart", [12, 24, 40])
@pytest.mark.parametrize("heads,kv,d,length", [(2, 1, 64, 17), (8, 2, 128, 18), (4, 1, 128, 33), (8, 1, 96, 146)])
def test_a_loud_block_behind_a_query(heads, kv, d, length, apart, dtype):
    """The newest position, or the newest two, begin a block of values 2^apart times the others', which the queries in front of
    them do not see."""
    table, pages = table_of([length], 16, 1)
    cache = cache_of(pages, kv, 16, d, 2)
    cache.v_scales.mul_(2.0 ** -8)
    q = torch.randn((1, 3, heads, d), generator=gen(3), device="cuda").to(dtype)
    cache.v_scales[table[0, (length - 1) // 16].long()] *= 2.0 ** apart
    got = ops.attention_cache_s8(q, cache, table, ints([length]))
    front = 3 - length % 16
    check(got[:, :front], q[:, :front], cache, table, [length - 3 + front], 16)
    if apart < 20:  # (its results hold these values)
        check(got, q, cache, table, [length], 16)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("length,loud", [(200, 5), (200, 0), (5000, 100)])
def test_rows_that_share_a_tile_and_look_at_unlike_blocks(length, loud, dtype):
    """Half of the heads look at the loud block alone, the other half not at all."""
    table, pages = table_of([length], 16, 1)
    cache = cache_of(pages, 1, 16, 128, 2)
    cache.v_scales.mul_(2.0 ** -14)
    q = torch.randn((1, 1, 8, 128), generator=gen(3), device="cuda").to(dtype)
    q[0, 0, ::2] = q[0, 0, 0]
    q[0, 0, 1::2] = -q[0, 0, 0]
    cache.v_scales[table[0, loud].long()] *= 2.0 ** 26
    against(cache, table, 0, loud * 16, q[0, 0], -60 * math.log(2))
    got = ops.attention_cache_s8(q[:, 0].contiguous(), cache, table, ints([length]))
    check(got[:, None], q, cache, table, [length], 16)


@pytest.mark.parametrize("spread", [10, 60])
def test_scales_of_all_sizes(spread):
    """Scales of values from 2^-spread to 2^spread, and small ones."""
    for lengths, queries, heads, d in (([700], 1, 8, 64), ([300, 50], 2, 16, 128), ([3000], 4, 4, 128)):
        table, pages = table_of(lengths, 16, 1)
        cache = cache_of(pages, 1, 16, d, 2)
        powers = torch.randint(-spread, spread + 1, cache.v_scales.shape, generator=gen(5), device="cuda")
        cache.v_scales.mul_(torch.ldexp(torch.ones_like(cache.v_scales), powers))
        q = 3 * torch.randn((len(lengths), queries, heads, d), generator=gen(3), device="cuda").bfloat16()
        check(ops.attention_cache_s8(q, cache, table, ints(lengths)), q, cache, table, lengths, 16)
        cache.v_scales.mul_(2.0 ** (spread - 90))
        check(ops.attention_cache_s8(q, cache, table, ints(lengths)), q, cache, table, lengths, 16)


def test_a_position_of_no_probability_whose_values_are_none():
    """0 times a NaN is one: every query that sees the block has it, however small its probability."""
    table, pages = table_of([100], 16, 1)
    for block, score in ((0, -200.0), (3, -200.0), (6, -200.0), (3, 1.0)):
        cache = cache_of(pages, 1, 16, 64, 2)
        q = torch.randn((1, 1, 64), generator=gen(3), device="cuda").bfloat16()
        against(cache, table, 0, block * 16, q[0], score)
        cache.v_scales[table[0, block].long()] = float("nan")
        assert bool(torch.isnan(ops.attention_cache_s8(q, cache, table, ints([100]))).all())


def test_values_next_to_the_largest():
    """An average of large values is none larger, whatever their number."""
    table, pages = table_of([4000], 16, 1)
    cache = cache_of(pages, 1, 16, 64, 2)
    cache.v.copy_(cache.v.abs().clamp(min=100))
    cache.v_scales.fill_(2.0 ** 120 * 0.99)
    q = torch.randn((1, 1, 4, 64), generator=gen(3), device="cuda").bfloat16()
    check(ops.attention_cache_s8(q[:, 0].contiguous(), cache, table, ints([4000]))[:, None], q, cache, table, [4000], 16)


@pytest.mark.parametrize("heads,kv,d", [(8, 1, 64), (16, 1, 128), (3, 1, 80)])
def test_queries_of_all_sizes(heads, kv, d):
    """Rows from the smallest numbers of bf16 to the largest, with keys that bring their scores to size."""
    table, pages = table_of([300], 16, 1)
    for e in (-126, -117, -106, -90, -20, 20, 100, 119, 120, 121, 122, 123, 124, 125, 126, 127):
        cache = cache_of(pages, kv, 16, d, 2)
        q = torch.rand((1, 1, heads, d), generator=gen(3), device="cuda") - 0.5
        q[0, 0, :, 0] = torch.linspace(1, 1.984375, heads, device="cuda")
        q = (q.double() * 2.0 ** e).bfloat16()
        assert bool(torch.isfinite(q).all())
        scale = 2.0 ** (-e / 2) / 3
        cache.k_scales.mul_(2.0 ** (-e - round(-e / 2)))
        got = ops.attention_cache_s8(q[:, 0].contiguous(), cache, table, ints([300]), scale=scale)
        check(got[:, None], q, cache, table, [300], 16, scale)


@pytest.mark.parametrize("over", [1, 2, 3, 4, 20, 2 ** 31 - 1 - 64])
def test_several_queries_of_a_sequence_longer_than_its_table(over):
    """Positions that the table has no room for are not seen; the others are by every query that comes behind them."""
    for heads, d in ((4, 64), (1, 128), (24, 64)):
        table, pages = table_of([64, 30], 16, 1)
        table = table[:, :4].contiguous()
        cache = cache_of(pages, 1, 16, d, 2)
        q = torch.randn((2, 4, heads, d), generator=gen(3), device="cuda").half()
        got = ops.attention_cache_s8(q, cache, table, ints([64 + over, 30]))
        torch.cuda.synchronize()
        assert ops.device_status() == 0x201
        check(got, q, cache, table, [64 + over, 30], 16)


def test_unused_slots_of_more_than_two_to_the_31_elements():
    """Their results are zeros to the last one."""
    cache = ops.kv_cache_s8(1, 1, 16, 128)
    queries, heads = 16385, 1024
    q = torch.zeros((1, 1, 1, 128), device="cuda").half().expand(1, queries, heads, 128)
    out = torch.full((1, queries, heads, 128), 7.0, dtype=torch.float16, device="cuda")
    ops.attention_cache_s8(q, cache, ints([[0]]), ints([0]), out=out)
    assert not bool(out.view(torch.int32).any())
    # two slots, one of them in use
    few = torch.full((2, 40, 64, 128), 7.0, dtype=torch.float16, device="cuda")
    ops.attention_cache_s8(q[:, :40, :64].expand(2, 40, 64, 128), cache, ints([[0], [0]]), ints([-1, 16]), out=few)
    assert not bool(few.any())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("length", [1, 3])
def test_probabilities_have_the_bits_that_results_need(length, dtype):
    """With a position or three the result is their values themselves, off by what probabilities are rounded to: fp16 results
    leave room for less than a single fp16 probability."""
    table, pages = table_of([length], 16, 1)
    for seed in range(20):
        cache = cache_of(pages, 2, 16, 64, seed)
        q = torch.randn((1, 1, 8, 64), generator=gen(seed), device="cuda").to(dtype)
        got = ops.attention_cache_s8(q[:, 0].contiguous(), cache, table, ints([length]))
        check(got[:, None], q, cache, table, [length], 16)

@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lengths,queries,heads,kv,d,page", [c for c in CASES if sum(c[0]) * c[2] < 20000])
def test_attention_within_the_bits_that_it_holds(lengths, queries, heads, kv, d, page, dtype):
    table, pages = table_of(lengths, page, 1)
    cache = cache_of(pages, kv, page, d, 2)
    q = torch.randn((len(lengths), queries, heads, d), generator=gen(3), device="cuda").to(dtype)
    got = ops.attention_cache_s8(q if queries > 1 else q[:, 0].contiguous(), cache, table, ints(lengths))
    check(got.view(q.shape), q, cache, table, lengths, page)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_queries_have_more_bits_than_their_type(dtype):
    """A row with one large element, where the keys have zeros: what the scores come from lies far below it."""
    table, pages = table_of([50], 16, 1)
    for down in (2.0 ** -6, 2.0 ** -9, 2.0 ** -11):
        cache = cache_of(pages, 1, 16, 64, 2)
        cache.k[..., 0] = 0
        q = torch.randn((1, 1, 8, 64), generator=gen(3), device="cuda")
        q[..., 0] = 1.5 / down
        q = q.to(dtype)
        got = ops.attention_cache_s8(q[:, 0].contiguous(), cache, table, ints([50]))
        check(got[:, None], q, cache, table, [50], 16)
