"""Attention over whole prompts against the definition in 64 bits, and the operators of a decoder's attention together."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_kv_cache import IDS, TYPES, angles, gen, ints, rows_at, sums, table_of, turned  # noqa: E402


def definition(q, k, v, counts, keys, causal, scale=None):
    """(out, how far the kernel's may be from it), packed.

    Roundings. A score: products of 16-bit numbers are exact, their sum over d is cut off at each step: (d + 8) 2^-23
    sum |q||k|. Its factor and the difference from the maximum, 3 2^-24 |t| each, and the power: 2^-22, or 2^-13.7 where the
    FMA pipe computes it for bf16 (2^-18.5 for fp16). P to its type: half a step, or for fp16 half of its smallest
    number of 2^6 times the probability: 2^-31 each. Sums over n keys, cut off: (n / 16 + 300) 2^-23. Twice what the powers have,
    for sum and total. The result: half a step of its type."""
    d, group = q.shape[2], q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    power = 2.0 ** -13.7 if q.dtype == torch.bfloat16 else 2.0 ** -18.5
    outs, offs = [], []
    for x, keys_, values in zip(q.double().split(counts), k.double().split(keys), v.double().split(keys)):
        n, m = x.shape[0], keys_.shape[0]
        out, off = torch.zeros_like(x), torch.zeros_like(x)
        for h in range(x.shape[1]):
            a, b, c = x[:, h], keys_[:, h // group], values[:, h // group]
            if m == 0 or n == 0:
                continue
            t = a @ b.t() * scale
            seen = torch.ones_like(t, dtype=torch.bool)
            if causal:
                seen = seen.tril(m - n)
            t = t.masked_fill(~seen, -math.inf)
            top = t.amax(1, keepdim=True)
            p = torch.exp(t - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = p.sum(1, keepdim=True)
            size = ((a.abs() @ b.abs().t()) * abs(scale)).masked_fill(~seen, 0)
            error = ((d + 8) * 2.0 ** -23 * size + 9 * 2.0 ** -24 * size).amax(1, keepdim=True) + 2.0 ** -22 + power
            relative = eps / 2 + 2 * torch.expm1(error.clamp(max=50)) + (m / 16 + 300) * 2.0 ** -23
            safe = torch.where(total == 0, torch.ones_like(total), total)
            out[:, h] = p @ c / safe
            off[:, h] = (p @ c.abs() / safe) * relative + (total > 0) * m * 2.0 ** -30 * c.abs().max()
        outs.append(out)
        offs.append((off + out.abs() * eps / 2 + torch.finfo(q.dtype).tiny * eps) * 1.001)
    return torch.cat(outs), torch.cat(offs)


def check(got, q, k, v, counts, keys, causal, scale=None):
    want, off = definition(q, k, v, counts, keys, causal, scale)
    far = (got.double() - want).abs() / off
    assert got.dtype == q.dtype and got.shape == q.shape
    assert bool((far <= 1).all()), (float(far.max()), int((far > 1).sum()))


def operands(counts, keys, heads, kv, d, dtype, seed=3):
    g = gen(seed)
    q = torch.randn((sum(counts), heads, d), generator=g, device="cuda")
    k, v = torch.randn((2, sum(keys), kv, d), generator=g, device="cuda")
    return q.to(dtype), k.to(dtype), (v + 0.5).to(dtype)


CASES = [  # queries, keys (None: alike), heads, kv, d, causal
    ([1], None, 1, 1, 16, True), ([2], None, 2, 1, 128, True), ([77], None, 8, 8, 64, True), ([127], None, 2, 2, 128, True),
    ([128], None, 4, 2, 128, True), ([129], None, 2, 1, 128, True), ([256], None, 2, 2, 64, True),
    ([257], None, 3, 3, 80, True), ([1000], None, 4, 1, 128, True), ([2049], None, 2, 2, 96, True),
    ([5, 0, 300, 1, 128, 40], None, 4, 2, 128, True), ([33] * 40, None, 2, 1, 32, True), ([511, 513], None, 5, 1, 112, True),
    ([77], None, 2, 2, 48, False), ([300, 20], None, 4, 4, 128, False), ([1024], None, 2, 1, 64, False),
    ([10, 200, 1], [400, 200, 129], 4, 2, 128, True), ([130], [1000], 2, 2, 64, True), ([300], [128], 2, 1, 128, True),
    ([300, 5], [0, 3], 2, 1, 64, True), ([20], [300], 2, 1, 128, False), ([4, 600], [0, 1300], 2, 2, 128, False),
    ([3000], None, 2, 1, 128, True), ([256 * 7], [256 * 7 + 64], 1, 1, 128, True),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("counts,keys,heads,kv,d,causal", CASES, ids=range(len(CASES)))
def test_attention(counts, keys, heads, kv, d, causal, dtype):
    m = keys or counts
    q, k, v = operands(counts, m, heads, kv, d, dtype)
    cu_k = None if keys is None else sums(keys)
    got = ops.attention_prompt(q, k, v, sums(counts), cu_k, causal=causal)
    check(got, q, k, v, counts, m, causal)
    assert ops.device_status() == 0
    assert torch.equal(got, ops.attention_prompt(q, k, v, sums(counts), cu_k, causal=causal))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5, 1e-3])
def test_scales_of_scores(scale, dtype):
    q, k, v = operands([400], [400], 2, 1, 128, dtype)
    check(ops.attention_prompt(q, k, v, sums([400]), scale=scale), q, k, v, [400], [400], True, scale)


@pytest.mark.parametrize("causal", [True, False])
def test_a_maximum_that_rises_all_the_way(causal):
    """Every tile of keys has larger scores than the one in front: sums are scaled each time."""
    q, k, v = operands([1200], [1200], 2, 1, 64, torch.bfloat16)
    q, k = q.abs(), k.abs()
    k *= torch.linspace(0.02, 4, 1200, device="cuda").bfloat16()[:, None, None]
    check(ops.attention_prompt(q, k, v, sums([1200]), causal=causal), q, k, v, [1200], [1200], causal)
    k = k.flip(0).contiguous()
    check(ops.attention_prompt(q, k, v, sums([1200]), causal=causal), q, k, v, [1200], [1200], causal)


def test_bad_values_reach_who_sees_them_only():
    counts = [300, 200, 61]
    q, k, v = operands(counts, counts, 2, 1, 64, torch.bfloat16)
    want = ops.attention_prompt(q, k, v, sums(counts))
    bad_k, bad_v, bad_q = k.clone(), v.clone(), q.clone()
    bad_v[250, 0, 7] = float("nan")   # seen by queries from 250 on
    bad_k[299, 0, 3] = float("inf")
    bad_k[300 + 130, 0, 0] = float("nan")
    bad_v[300 + 199, 0, 1] = float("-inf")
    bad_q[520, 1, 5] = float("nan")
    got = ops.attention_prompt(bad_q, bad_k, bad_v, sums(counts))
    clean = torch.ones((561, 2), dtype=torch.bool, device="cuda")
    clean[250:300], clean[430:500], clean[520, 1] = False, False, False
    assert torch.equal(got[:128], want[:128]) and torch.equal(got[500:520], want[500:520])
    off = definition(q, k, v, counts, counts, True)[1]
    assert bool(((got.double() - want.double()).abs()[clean] <= 2 * off[clean]).all())
    assert bool(torch.isnan(got[250:300, :, 7]).all()) and bool(torch.isfinite(got[250:299, :, :7]).all())
    assert bool(torch.isnan(got[430:500]).all()) and bool(torch.isnan(got[520, 1]).all())


@pytest.mark.parametrize("filler", [float("nan"), float("inf")])
def test_rows_behind_the_last_sequence(filler):
    """A padded batch: the padding holds anything, and its rows of the result are left as they were."""
    q, k, v = operands([700], [700], 4, 2, 128, torch.float16)
    want = ops.attention_prompt(q[:203], k[:203], v[:203], sums([40, 163]))
    for x in (q, k, v):
        x[203:] = filler
    out = torch.full_like(q, 7)
    got = ops.attention_prompt(q, k, v, ints([0, 40, 203]), out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out[:203], want) and bool((out[203:] == 7).all())


def test_strides_and_orders():
    """Slices of one projection; heads in front of tokens; a result with gaps."""
    counts = [150, 90]
    qkv = torch.randn((240, 8, 128), generator=gen(3), device="cuda").half()
    q, k, v = qkv.split((4, 2, 2), 1)
    want = ops.attention_prompt(q.contiguous(), k.contiguous(), v.contiguous(), sums(counts))
    assert torch.equal(ops.attention_prompt(q, k, v, sums(counts)), want)
    turned_round = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(ops.attention_prompt(*turned_round, sums(counts)), want)
    out = torch.full((240, 5, 150), 7.0, device="cuda").half()
    ops.attention_prompt(q, k, v, sums(counts), out=out[:, :4, 3:131])
    assert torch.equal(out[:, :4, 3:131], want)
    out[:, :4, 3:131] = 7
    assert bool((out == 7).all())


def test_units_that_the_loads_cannot_take_are_refused():
    from megcc_b200._lib import MegccError
    flat = torch.zeros(100 * 4 * 72, device="cuda").half()
    for view in (flat[1:1 + 90 * 4 * 64].view(90, 4, 64), flat[:90 * 4 * 68].view(90, 4, 68)[..., :64]):
        good = torch.zeros((90, 4, 64), device="cuda").half()
        with pytest.raises(MegccError):
            ops.attention_prompt(view, good, good, sums([90]))
        with pytest.raises(MegccError):
            ops.attention_prompt(good, good, view, sums([90]))


def test_captured_and_on_two_streams():
    q, k, v = operands([300], [300], 4, 2, 64, torch.bfloat16)
    cu, out = ints([0, 100, 300]), torch.zeros_like(q)
    ops.attention_prompt(q, k, v, cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_prompt(q, k, v, cu, out=out)
    for lengths in ([0, 100, 300], [0, 299, 300], [0, 0, 7]):
        cu.copy_(ints(lengths))
        out.zero_()
        graph.replay()
        assert torch.equal(out, ops.attention_prompt(q, k, v, cu, out=torch.zeros_like(q)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    cu.copy_(ints([0, 100, 300]))
    want = ops.attention_prompt(q, k, v, cu)
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.attention_prompt(q, k, v, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_decoder_s_attention():
    """Prompts into an empty cache, a second part that continues them over what is cached, then tokens one by one: each
    query's result is the attention over all positions in front of it, as far as the cache's rounding goes: a value is
    half a step of its block's scale off at most, and half a step more for each time that the scale grew."""
    heads, kv, d, page, dtype = 4, 2, 64, 32, torch.bfloat16
    first, second, steps = [70, 130], [40, 9], 3
    total = [a + b + steps for a, b in zip(first, second)]
    table, pages = table_of(total, page, 5)
    cache, (cos, sin) = ops.kv_cache_s8(pages, kv, page, d), angles(200, d)
    q, k, v = operands(total, total, heads, kv, d, dtype)
    at = [0, total[0]]
    position = torch.cat([torch.arange(t) for t in total]).cuda()
    qt, kt = (turned(x, cos, sin, position, False).to(dtype) for x in (q, k))
    want, off = definition(qt, kt, v, total, total, True)

    def rows(x, start, n):
        return torch.cat([x[a + s:a + s + c] for a, s, c in zip(at, start, n)])

    def far(got, start, n):
        """in units of the bound: p's error is that of a score, |q| times half a step of each key (8 in all, times the growth
        of the scale), V's is its own"""
        step = float(max(cache.k_scales.max(), cache.v_scales.max())) * 8.5
        score = float(qt.float().abs().sum(-1).max()) / math.sqrt(d) * step / 8.5 * 0.5
        return ((got.double() - rows(want, start, n)).abs() / (rows(off, start, n) + step + math.expm1(2 * score) * 3.5)).max()

    zero = [0, 0]
    q1, k1 = ops.kv_append_s8(cache, table, ints(zero), rows(k, zero, first), rows(v, zero, first), rows(q, zero, first),
                              cos, sin, cu_tokens=sums(first), turned_keys=True)
    out = ops.attention_prompt(q1, k1, rows(v, zero, first), sums(first))
    check(out, q1, k1, rows(v, zero, first), first, first, True)
    assert torch.equal(k1, rows(kt, zero, first)) and torch.equal(q1, rows(qt, zero, first))
    q2, _ = ops.kv_append_s8(cache, table, ints(first), rows(k, first, second), rows(v, first, second),
                             rows(q, first, second), cos, sin, cu_tokens=sums(second))
    held = [a + b for a, b in zip(first, second)]
    keys, values = ops.kv_read_s8(cache, table, None, sums(held), sum(held), dtype)
    out = ops.attention_prompt(q2, keys, values, sums(second), sums(held))
    check(out, q2, keys, values, second, held, True)
    assert far(out, first, second) < 1
    for s in range(steps):
        now = [h + s for h in held]
        q3, _ = ops.kv_append_s8(cache, table, ints(now), rows(k, now, [1, 1]), rows(v, now, [1, 1]),
                                 rows(q, now, [1, 1]), cos, sin)
        out = ops.attention_cache_s8(q3, cache, table, ints([n + 1 for n in now]))
        assert far(out, now, [1, 1]) < 1
        # the same by reading back
        keys, values = ops.kv_read_s8(cache, table, None, sums([n + 1 for n in now]), sum(now) + 2, dtype)
        check(ops.attention_prompt(q3, keys, values, sums([1, 1]), sums([n + 1 for n in now])), q3, keys, values, [1, 1],
              [n + 1 for n in now], True)
    assert ops.device_status() == 0
