"""The int8 cache of keys and values: appending with the position rotation, reading back, against the definition.
Every step of it is one rounding (a quotient of 24-bit numbers that is no tie is further from one than 64 bits' rounding), so
whole numbers, scales and values have to be equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402

TYPES = [torch.float16, torch.bfloat16]
IDS = ["f16", "bf16"]
BLOCK = 16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def sums(v):
    got = [0]
    for n in v:
        got.append(got[-1] + n)
    return ints(got)


def cache_of(pages, kv, page, d, seed):
    shape, blocks = (pages, kv, page, d), (pages, kv, page // BLOCK)
    g = gen(seed)
    return ops.KvCacheS8(*(torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in "kv"),
                         *(torch.rand(blocks, generator=g, device="cuda") * 0.02 + 0.005 for _ in "kv"))


def table_of(held, page, seed, spare=2):
    """Pages in any order; -1 where a sequence has none."""
    need = [-(-h // page) for h in held]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(held), max(need + [1]) + 1), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table.cuda(), sum(need) + spare


def angles(positions, rot, seed=3):
    a = torch.rand((positions, rot // 2), generator=gen(seed), device="cuda") * 6.28
    return a.cos(), a.sin()


def turned(x, cos, sin, position, interleaved):
    """fp32, products and sums rounded each (every operation is a kernel of its own here)"""
    rot, x = 2 * cos.shape[1], x.float()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    c, s = cos[position][:, None], sin[position][:, None]
    p, q, y = x[..., first], x[..., second], x.clone()
    pc, qs, qc, ps = p * c, q * s, q * c, p * s
    y[..., first], y[..., second] = pc - qs, qc + ps
    return y


def block_scale(amax):
    s = (amax.double().clamp(min=2.0 ** -119) / 127).float()
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))


def whole_of(x):
    """64 bits to the nearest whole number; what is none counts 0"""
    q = torch.round(x)
    return torch.where(torch.isfinite(q), q, torch.zeros_like(q)).to(torch.int8)


def append_definition(whole, scales, table, before, counts, x, page):
    """x: fp32 [tokens, heads, d], appended to one tensor of the cache in place"""
    row = 0
    for b, (c, n) in enumerate(zip(before, counts)):
        p, end, at = c, c + n, row
        row += n
        while c >= 0 and p < end:
            first = p // BLOCK * BLOCK
            last = min(first + BLOCK, end)
            number, o = int(table[b, first // page]), first % page
            new = x[at:at + last - p]
            amax = new.abs().amax((0, 2))
            amax = torch.where(torch.isnan(new).any(-1).any(0), torch.full_like(amax, float("nan")), amax)
            s, old = block_scale(amax), scales[number, :, o // BLOCK].clone()
            if p > first:
                s = torch.where(torch.isnan(s) | torch.isnan(old), s + old, torch.maximum(s, old))
                kept = whole[number, :, o:o + p - first]
                again = whole_of(kept.double() * (old.double() / s.double())[:, None, None])
                whole[number, :, o:o + p - first] = torch.where((s == old)[:, None, None], kept, again)
            quotient = new.transpose(0, 1).double() / s.double()[:, None, None]
            whole[number, :, o + p - first:o + last - first] = whole_of(quotient)
            scales[number, :, o // BLOCK] = s
            at, p = at + last - p, last


def same_scales(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def rows_at(cache, table, b, n, page, dtype):
    """Values of the first n positions of sequence b: ([n, heads, d] of keys, of values)"""
    p = torch.arange(n, device="cuda")
    number, o = table[b, p // page].long(), p % page
    return [(w[number, :, o].float() * s[number, :, o // BLOCK][..., None]).to(dtype) for w, s in
            ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]


CASES = [  # before, counts, heads, kv, d, rot, page, interleaved
    ([0], [1], 1, 1, 16, 16, 16, False),
    ([15], [1], 4, 2, 128, 128, 64, False),
    ([16], [1], 3, 3, 64, 32, 16, True),
    ([5, 16, 31, 0, 100], [1] * 5, 8, 2, 128, 128, 32, False),
    ([0], [16], 2, 1, 64, 64, 16, False),
    ([3], [45], 5, 5, 80, 48, 32, True),
    ([0, 14, 7, 250, 32], [17, 0, 1, 130, 33], 6, 2, 112, 112, 64, False),
    ([1, 2, 3], [2, 18, 14], 40, 1, 48, 16, 48, False),
    ([63, 65, -1, 9], [2, 31, 3, 0], 4, 4, 96, 96, 64, True),
    (list(range(40)), [1 + i % 3 for i in range(40)], 2, 1, 32, 32, 16, False),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("before,counts,heads,kv,d,rot,page,interleaved", CASES, ids=range(len(CASES)))
def test_append(before, counts, heads, kv, d, rot, page, interleaved, dtype):
    n = sum(counts)
    held = [max(0, c) + m for c, m in zip(before, counts)]
    table, pages = table_of(held, page, 1)
    cache = cache_of(pages, kv, page, d, 2)
    want = ops.KvCacheS8(*(t.clone() for t in cache))
    cos, sin = angles(max(held) + 1, rot)
    qkv = torch.randn((n, heads + 2 * kv, d), generator=gen(4), device="cuda").to(dtype)
    q, k, v = qkv.split((heads, kv, kv), 1)
    one = counts == [1] * len(counts)
    got_q, got_k = ops.kv_append_s8(cache, table, ints(before), k, v, q, cos, sin, interleaved=interleaved,
                                    cu_tokens=None if one else sums(counts), turned_keys=True)
    position = torch.tensor([max(0, c) + i for c, m in zip(before, counts) for i in range(m)], device="cuda")
    used = torch.tensor([c >= 0 for c, m in zip(before, counts) for _ in range(m)], device="cuda")
    qt, kt = (turned(x, cos, sin, position, interleaved) for x in (q, k))
    assert torch.equal(got_q[used], qt.to(dtype)[used]) and torch.equal(got_k[used], kt.to(dtype)[used])
    append_definition(want.k, want.k_scales, table, before, counts, kt, page)
    append_definition(want.v, want.v_scales, table, before, counts, v.float(), page)
    # (positions behind the last new one count for nothing)
    for b, (c, m) in enumerate(zip(before, counts)):
        if c >= 0:
            for x, y in zip(rows_at(cache, table, b, c + m, page, torch.float32),
                            rows_at(want, table, b, c + m, page, torch.float32)):
                assert torch.equal(x, y), b
    assert torch.equal(cache.k_scales, want.k_scales) and torch.equal(cache.v_scales, want.v_scales)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_quotients_in_the_middle_and_next_to_it(dtype):
    """Whole multiples of a number: quotients by the scale that are ties, or within a rounding of one."""
    table, pages = table_of([64], 64, 1)
    for unit in (1.0, 0.75, 2.0 ** -20, 1.5 * 2.0 ** -90 if dtype == torch.bfloat16 else 3.0):
        for most in (127, 254, 85, 170, 255, 100):
            cache = cache_of(pages, 1, 64, 128, 2)
            want = ops.KvCacheS8(*(t.clone() for t in cache))
            x = torch.randint(-most, most + 1, (64, 1, 128), generator=gen(most), device="cuda")
            x[:, 0, 0] = most
            x = (x.double() * unit).to(dtype)
            ops.kv_append_s8(cache, table, ints([0]), x, -x, cu_tokens=ints([0, 64]))
            append_definition(want.k, want.k_scales, table, [0], [64], x.float(), 64)
            append_definition(want.v, want.v_scales, table, [0], [64], -x.float(), 64)
            assert torch.equal(cache.k[table[0, 0].long()], want.k[table[0, 0].long()]), (unit, most)
            assert all(torch.equal(a, b) for a, b in zip(cache, want)), (unit, most)


def test_append_without_rotation_and_queries():
    table, pages = table_of([21], 32, 1)
    cache = cache_of(pages, 2, 32, 64, 2)
    want = ops.KvCacheS8(*(t.clone() for t in cache))
    k, v = torch.randn((2, 5, 2, 64), generator=gen(3), device="cuda").half()
    assert ops.kv_append_s8(cache, table, ints([16]), k, v, cu_tokens=ints([0, 5])) == (None, None)
    append_definition(want.k, want.k_scales, table, [16], [5], k.float(), 32)
    append_definition(want.v, want.v_scales, table, [16], [5], v.float(), 32)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


@pytest.mark.parametrize("offset", [0, 1, 3])
def test_operands_at_any_element_and_pitch(offset):
    def at(shape, pitch, seed):
        t, h, d = shape
        flat = torch.randn(offset + t * h * pitch + 64, generator=gen(seed), device="cuda").bfloat16()
        return flat.as_strided(shape, (h * pitch, pitch, 1), offset)
    table, pages = table_of([40], 16, 1)
    caches = [cache_of(pages, 2, 16, 64, 2) for _ in range(2)]
    cos, sin = angles(40, 64)
    q, k, v = at((17, 4, 64), 67, 3), at((17, 2, 64), 65, 4), at((17, 2, 64), 64, 5)
    odd = ops.kv_append_s8(caches[0], table, ints([20]), k, v, q, cos, sin, cu_tokens=ints([0, 17]), turned_keys=True)
    plain = ops.kv_append_s8(caches[1], table, ints([20]), k.contiguous(), v.contiguous(), q.contiguous(), cos, sin,
                             cu_tokens=ints([0, 17]), turned_keys=True)
    assert all(torch.equal(a, b) for a, b in zip(odd + tuple(caches[0]), plain + tuple(caches[1])))


def test_a_token_at_a_time_is_what_the_definition_says():
    table, pages = table_of([37], 16, 5)
    cache = cache_of(pages, 3, 16, 32, 2)
    want = ops.KvCacheS8(*(t.clone() for t in cache))
    for p in range(37):
        x = (torch.randn((1, 3, 32), generator=gen(p), device="cuda") * (1 + p % 5)).half()
        ops.kv_append_s8(cache, table, ints([p]), x, -x)
        append_definition(want.k, want.k_scales, table, [p], [1], x.float(), 16)
        append_definition(want.v, want.v_scales, table, [p], [1], -x.float(), 16)
    for x, y in zip(rows_at(cache, table, 0, 37, 16, torch.float32), rows_at(want, table, 0, 37, 16, torch.float32)):
        assert torch.equal(x, y)


def test_infinities_and_nans_stay_in_their_block_and_head():
    table, pages = table_of([40], 16, 1)
    cache = cache_of(pages, 2, 16, 32, 2)
    k = torch.randn((40, 2, 32), generator=gen(3), device="cuda").bfloat16()
    v = k.clone()
    k[3, 0, 5], v[17, 1, 0], v[18, 1, 0] = float("nan"), float("inf"), float("-inf")
    ops.kv_append_s8(cache, table, ints([0]), k, v, cu_tokens=ints([0, 40]))
    kr, vr = ops.kv_read_s8(cache, table, None, ints([0, 40]), 40)
    bad_k, bad_v = torch.isnan(kr), torch.isnan(vr)
    assert bad_k[:16, 0].all() and not bad_k[16:].any() and not bad_k[:, 1].any()
    assert bad_v[16:32, 1].all() and int(bad_v.sum()) == 16 * 32
    # ... as long as the block keeps them: appended to, and begun anew
    fresh = torch.ones((1, 2, 32), device="cuda").bfloat16()
    ops.kv_append_s8(cache, table, ints([4]), fresh, fresh)
    assert torch.isnan(ops.kv_read_s8(cache, table, None, ints([0, 5]), 5)[0][:, 0]).all()
    ops.kv_append_s8(cache, table, ints([0]), fresh, fresh)
    assert torch.equal(ops.kv_read_s8(cache, table, None, ints([0, 1]), 1)[0], fresh)


def test_zeros_and_the_smallest_values():
    table, pages = table_of([32], 16, 1)
    cache = cache_of(pages, 1, 16, 16, 2)
    x = torch.zeros((32, 1, 16), device="cuda").bfloat16()
    x[20] = 2.0 ** -130
    ops.kv_append_s8(cache, table, ints([0]), x, x, cu_tokens=ints([0, 32]))
    kr, _ = ops.kv_read_s8(cache, table, None, ints([0, 32]), 32)
    assert bool((kr == 0).all()) and bool((cache.k_scales > 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("starts,counts,kv,d,page", [
    ([0], [1], 1, 16, 16), ([7], [30], 2, 128, 16), (None, [100, 3, 0, 41], 3, 80, 32), ([5, 0, 64], [17, 64, 1], 8, 64, 64),
    ([0] * 40, [1 + i % 4 for i in range(40)], 1, 112, 48), ([4090], [33], 4, 128, 128)])
def test_read(starts, counts, kv, d, page, dtype):
    from_ = starts or [0] * len(counts)
    table, pages = table_of([s + n for s, n in zip(from_, counts)], page, 3)
    cache = cache_of(pages, kv, page, d, 4)
    n = sum(counts)
    k, v = ops.kv_read_s8(cache, table, None if starts is None else ints(starts), sums(counts), n, dtype)
    row = 0
    for b, (s, m) in enumerate(zip(from_, counts)):
        want_k, want_v = rows_at(cache, table, b, s + m, page, dtype)
        assert torch.equal(k[row:row + m], want_k[s:]) and torch.equal(v[row:row + m], want_v[s:])
        row += m
    assert ops.device_status() == 0


def test_rows_of_no_sequence_are_left_as_they_were():
    """Through the C entry, whose results the caller brings: rows behind the last sequence, and in front of the first."""
    import ctypes as C
    from megcc_b200 import _lib
    table, pages = table_of([20, 20], 16, 3)
    cache = cache_of(pages, 2, 16, 32, 4)
    c = _lib.KvCache(cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scales.data_ptr(), cache.v_scales.data_ptr(),
                     table.data_ptr(), table.stride(0), pages, 2, 16, 32, 2, table.shape[1])
    k, v = torch.full((2, 50, 2, 32), 7.0, device="cuda").half()
    cu = ints([3, 20, 30])
    heads = [_lib.Heads(t.data_ptr(), 64, 32) for t in (k, v)]
    _lib.check(_lib.lib().mb200_kv_read_s8(C.byref(c), None, cu.data_ptr(), 50, 1, C.byref(heads[0]), C.byref(heads[1]),
                                           torch.cuda.current_stream().cuda_stream))
    for b, (first, n) in enumerate(((3, 17), (20, 10))):
        want = rows_at(cache, table, b, n, 16, torch.float16)
        assert torch.equal(k[first:first + n], want[0]) and torch.equal(v[first:first + n], want[1])
    for t in (k, v):
        assert bool((t[:3] == 7).all()) and bool((t[30:] == 7).all())
    before = [t.clone() for t in cache]
    x = torch.randn((50, 2, 32), generator=gen(1), device="cuda").half()
    lengths, h = ints([0, -1]), _lib.Heads(x.data_ptr(), 64, 32)
    out = _lib.Heads(k.data_ptr(), 64, 32)
    p = _lib.KvAppendParam(lengths.data_ptr(), cu.data_ptr(), 50, 0, 1, h, h, _lib.Heads(), _lib.Heads(), out, None, None,
                           0, 0, 0)
    k.fill_(5)
    _lib.check(_lib.lib().mb200_kv_append_s8(C.byref(c), C.byref(p), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(k[3:20], x[3:20]) and bool((k[:3] == 5).all()) and bool((k[20:] == 5).all())
    other = table[1, :2].long()  # (a sequence that is not in use)
    assert all(torch.equal(a[other], b[other]) for a, b in zip(cache, before))


def test_positions_without_a_page_are_reported():
    table, pages = table_of([16, 16], 16, 3)
    table[1, 0] = pages  # not in the pool
    cache = cache_of(pages, 1, 16, 16, 4)
    before = [t.clone() for t in cache]
    x = torch.ones((2, 1, 16), device="cuda").half()
    _, turned_k = ops.kv_append_s8(cache, table, ints([16, 3]), x, x, turned_keys=True)  # (table entries -1 and `pages`)
    assert torch.equal(turned_k, x)
    torch.cuda.synchronize()
    assert ops.device_status() == 0x201 and ops.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    k, v = ops.kv_read_s8(cache, table, ints([15, 10 ** 6]), ints([0, 3, 5]), 5, torch.float16)
    torch.cuda.synchronize()
    assert ops.device_status() == 0x201
    assert torch.equal(k[0], rows_at(cache, table, 0, 16, 16, torch.float16)[0][15])
    assert bool((k[1:] == 0).all()) and bool((v[1:] == 0).all())
    # beyond the rotation's tables
    cos, sin = angles(4, 16)
    _, turned_k = ops.kv_append_s8(cache, table, ints([4, -1]), x, x, None, cos, sin, turned_keys=True)
    torch.cuda.synchronize()
    assert ops.device_status() == 0x202 and bool(torch.isnan(turned_k[0]).all())


def test_a_captured_step_goes_by_the_lengths_it_finds():
    table, pages = table_of([64, 64], 16, 3)
    caches = [cache_of(pages, 2, 16, 64, 4) for _ in range(2)]
    lengths, cos, sin = ints([3, 30]), *angles(64, 64)
    qkv = torch.randn((2, 8, 64), generator=gen(3), device="cuda").half()
    q, k, v = qkv.split((4, 2, 2), 1)

    def step(cache):
        q2, _ = ops.kv_append_s8(cache, table, lengths, k, v, q, cos, sin)
        out = ops.attention_cache_s8(q2, cache, table, lengths + 1)
        lengths.add_(1)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache_of(pages, 2, 16, 64, 4))
    torch.cuda.current_stream().wait_stream(side)
    lengths.copy_(ints([3, 30]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0])
    got = []
    for i in range(20):
        qkv.copy_(torch.randn((2, 8, 64), generator=gen(10 + i), device="cuda"))
        graph.replay()
        got.append(captured.clone())
    lengths.copy_(ints([3, 30]))
    for i in range(20):
        qkv.copy_(torch.randn((2, 8, 64), generator=gen(10 + i), device="cuda"))
        assert torch.equal(step(caches[1]), got[i]), i
    assert all(torch.equal(a, b) for a, b in zip(*caches))
