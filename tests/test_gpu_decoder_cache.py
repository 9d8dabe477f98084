"""What a decoder gets from the int8 cache: prompts, prompts that continue, single tokens, in the order in which they are used."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_attention_cache_range import check  # noqa: E402
from test_gpu_attention_prompt import check as check_prompt  # noqa: E402
from test_gpu_kv_cache import BLOCK, IDS, TYPES, angles, gen, ints, rows_at, sums, table_of, turned  # noqa: E402


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 64, 32), (8, 1, 128, 16)])
def test_a_decoder_s_cache_and_results(heads, kv, d, page, dtype):
    """Each cached number is what was appended, half a step of its block's scale off, and half a step more for each later append
    to its block, which may make it anew; each result is the attention over what the cache holds, within the kernel's
    own bound. Both follow from the definitions, and together they leave the result no room."""
    first, second, steps = [70, 130], [40, 9], 20
    total = [a + b + steps for a, b in zip(first, second)]
    table, pages = table_of(total, page, 5)
    cache, (cos, sin) = ops.kv_cache_s8(pages, kv, page, d), angles(200, d)
    g = gen(3)
    q = torch.randn((sum(total), heads, d), generator=g, device="cuda").to(dtype)
    k, v = torch.randn((2, sum(total), kv, d), generator=g, device="cuda").add(0.5).to(dtype)
    at, position = [0, total[0]], torch.cat([torch.arange(t) for t in total]).cuda()
    kt = turned(k, cos, sin, position, False)  # (what the cache is made from)
    calls = [[] for _ in total]  # first position of each append

    def rows(x, start, n):
        return torch.cat([x[a + s:a + s + c] for a, s, c in zip(at, start, n)])

    def append(start, n):
        for c, s in zip(calls, start):
            c.append(s)
        one = n == [1] * len(n)
        return ops.kv_append_s8(cache, table, ints(start), rows(k, start, n), rows(v, start, n), rows(q, start, n), cos, sin,
                                cu_tokens=None if one else sums(n))[0]

    def check_cache(held):
        for b, n in enumerate(held):
            p = torch.arange(n, device="cuda")
            # appends that came behind a position's own and began in its block
            later = torch.zeros(n, dtype=torch.float64, device="cuda")
            for s in calls[b]:
                later += ((s // BLOCK == p // BLOCK) & (p < s)).double()
            got = rows_at(cache, table, b, n, page, torch.float64)
            for have, scales, true in zip(got, (cache.k_scales, cache.v_scales), (kt, v.float())):
                step = scales[table[b, p // page].long(), :, p % page // BLOCK].double()
                # (values in fp32: number times scale, rounded)
                bound = (0.5 * (1 + later))[:, None] * step * (1 + 2.0 ** -20) + 127 * step * 2.0 ** -24
                off = (have.double() - true[at[b]:at[b] + n].double()).abs().amax(-1)
                assert bool((off <= bound).all()), float((off / bound).max())

    zero = [0, 0]
    append(zero, first)
    check_cache(first)
    q2 = append(first, second)
    held = [a + b for a, b in zip(first, second)]
    check_cache(held)
    keys, values = ops.kv_read_s8(cache, table, None, sums(held), sum(held), dtype)
    check_prompt(ops.attention_prompt(q2, keys, values, sums(second), sums(held)), q2, keys, values, second, held, True)
    for s in range(steps):
        q3 = append([h + s for h in held], [1, 1])
        now = [h + s + 1 for h in held]
        check_cache(now)
        out = ops.attention_cache_s8(q3, cache, table, ints(now))
        check(out[:, None], q3[:, None], cache, table, now, page)
    assert ops.device_status() == 0


def test_what_the_cache_costs_a_decoder():
    """Results over the cache against those over the keys and values themselves. A number is off by step / sqrt(12) on average,
    and a block's step is its largest / 127: of 16 x 128 normal numbers the largest is 3.2 to 4.2 times their spread, so 0.007
    to 0.0095 of it. That is the part that values bring, and scores, off by |q| / sqrt(d) = 1 times as much, bring the same
    again: sum p dt (v - out) is as large as sum p dv. Together 0.010 to 0.0135 of the results' own size; 0.03 is twice that."""
    n, heads, kv, d, page = 1000, 8, 2, 128, 64
    table, pages = table_of([n], page, 5)
    cache = ops.kv_cache_s8(pages, kv, page, d)
    q = torch.randn((1, heads, d), generator=gen(1), device="cuda").bfloat16()
    k, v = torch.randn((2, n, kv, d), generator=gen(2), device="cuda").bfloat16()
    ops.kv_append_s8(cache, table, ints([0]), k, v, cu_tokens=ints([0, n]))
    got = ops.attention_cache_s8(q, cache, table, ints([n])).double()[0]
    wide_k, wide_v = (x.double().repeat_interleave(heads // kv, 1).transpose(0, 1) for x in (k, v))
    p = torch.softmax((wide_k @ q[0].double()[..., None])[..., 0] / math.sqrt(d), -1)
    want = (p[:, None] @ wide_v)[:, 0]
    rms = float((got - want).square().mean().sqrt() / want.square().mean().sqrt())
    assert rms < 0.03
