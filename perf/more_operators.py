"""Performance cases of attention with an int8 cache: keys and values appended to a paged cache with the
position rotation on the way, cached ones read back in 16 bits, attention over the cache for one or a few
queries per sequence, attention over whole prompts.

``listed()`` are fixed cases, ``draw()`` gives further ones of the same ranges; ``prepare`` makes what
a program holds before the call, ``run`` is one pass, ``work`` the bytes and operations the pass
cannot do without, ``exact`` its results in 64 bits. Where ``own`` is false ``run`` computes the plain
form from elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16           # positions of a head that share a scale
TINY = 2.0 ** -119   # the least magnitude a scale is taken from
GOLDEN = 0.6180339887498949


def _append(name, batch, tokens, cached, heads, kv, d, rot, page, dtype, interleaved=False):
    return dict(name=name, kind="append", batch=batch, tokens=tokens, cached=cached, heads=heads, kv=kv, d=d,
                rot=rot, page=page, dtype=dtype, interleaved=interleaved)


def _read(name, batch, tokens, kv, d, page, dtype):
    return dict(name=name, kind="read", batch=batch, tokens=tokens, kv=kv, d=d, page=page, dtype=dtype)


def _cache(name, batch, longest, queries, heads, kv, d, page, dtype, empty=0):
    return dict(name=name, kind="cache", batch=batch, longest=longest, queries=queries, heads=heads, kv=kv, d=d,
                page=page, dtype=dtype, empty=empty)


def _prompt(name, batch, tokens, prefix, heads, kv, d, dtype, causal=True):
    return dict(name=name, kind="prompt", batch=batch, tokens=tokens, prefix=prefix, heads=heads, kv=kv, d=d,
                dtype=dtype, causal=causal)


def listed():
    return [
        # One decoding step of one sequence: its token's keys and values, queries turned beside them.
        _append("append_t1", 1, 1, 500, 32, 8, 128, 128, 64, "bf16"),
        # A decoding step of an odd number of sequences; half of each head is turned, neighbours as pairs.
        _append("append_b61", 61, 61, 4000, 24, 4, 64, 32, 16, "f16", True),
        # Prompts of several sequences that continue what is cached, starting anywhere in a block.
        _append("append_prompt", 5, 8191, 2000, 32, 8, 128, 128, 64, "bf16"),
        # The cached prefix of one prompt, for the attention over the whole of it.
        _read("read_prefix", 1, 1000, 8, 128, 64, "bf16"),
        # Prefixes of a batch of prompts, ragged.
        _read("read_b16", 16, 65001, 8, 128, 32, "f16"),
        # One sequence, one token: latency counts.
        _cache("cache_b1", 1, 2047, 1, 32, 8, 128, 64, "bf16"),
        # One sequence over a very long context: all of the GPU on a few heads.
        _cache("cache_b1_long", 1, 131071, 1, 32, 8, 128, 64, "bf16"),
        # A decoding step of many sequences of unlike lengths, small pages, some slots of the batch unused.
        _cache("cache_b48", 48, 8192, 1, 32, 4, 128, 16, "f16", 3),
        # Checking four proposed tokens per sequence, a key head for each query head.
        _cache("cache_b8_verify", 8, 6001, 4, 16, 16, 64, 32, "bf16"),
        # A short prompt, one tile and odd.
        _prompt("prompt_t77", 1, 77, 0, 8, 8, 64, "f16"),
        # Prompts of several sequences, packed, of unlike odd lengths.
        _prompt("prompt_b9", 9, 4099, 0, 32, 8, 128, "bf16"),
        # A long prompt: bound by the tensor cores and the exponentials.
        _prompt("prompt_t8192", 1, 8192, 0, 32, 8, 128, "bf16"),
    ]


def _log(rng, low, high, multiple=1):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, v // multiple * multiple)


def draw(rng):
    kind = rng.choice(["append", "read", "cache", "cache", "prompt", "prompt"])
    dtype = rng.choice(["bf16", "f16"])
    d = rng.choice([64, 128, 128, 16 * rng.randint(2, 8)])
    page = rng.choice([16, 32, 64, 128])
    while True:
        kv = rng.choice([1, 2, 4, 8, 8, 16])
        heads = kv * rng.choice([1, 2, 4, 4, 5, 8])
        batch = _log(rng, 1, 128)
        if kind == "append":
            tokens = batch if rng.random() < 0.5 else max(batch, _log(rng, 16, 8191))
            rot = d if rng.random() < 0.6 else 16 * rng.randint(1, d // 16)
            if tokens * heads <= 8191 * 32:
                return dict(kind=kind, batch=batch, tokens=tokens, cached=_log(rng, 1, 8000), heads=heads, kv=kv, d=d,
                            rot=rot, page=page, dtype=dtype, interleaved=rng.random() < 0.3)
        elif kind == "read":
            tokens = max(batch, _log(rng, 16, 65001))
            if tokens * kv * d <= 65001 * 8 * 128:
                return dict(kind=kind, batch=batch, tokens=tokens, kv=kv, d=d, page=page, dtype=dtype)
        elif kind == "cache":
            longest = _log(rng, 1, 131071)
            queries = rng.choice([1, 1, 1, 2, 4, 7])
            if batch * longest * kv * d <= 48 * 8192 * 8 * 128 and batch * longest * queries * heads <= 48 * 8192 * 64:
                return dict(kind=kind, batch=batch, longest=longest, queries=queries, heads=heads, kv=kv, d=d,
                            page=page, dtype=dtype, empty=rng.choice([0, 0, batch // 4]))
        else:
            tokens = max(batch, _log(rng, 16, 8192))
            prefix = rng.choice([0, 0, _log(rng, 1, 2048)])
            # (the plain form pads every sequence to the longest, which is up to four times the mean)
            long = min(tokens, 4 * tokens // batch + 1)
            if heads <= 40 and batch * heads * long * (long + 2 * prefix) <= 32 * 8192 ** 2:
                return dict(kind=kind, batch=batch, tokens=tokens, prefix=prefix, heads=heads, kv=kv, d=d, dtype=dtype,
                            causal=rng.random() < 0.8)


# ---- lengths that follow from the case alone ----
def _shares(total, n):
    """n whole numbers of at least 1 with this sum, the largest several times the smallest."""
    if total == n:
        return [1] * n
    weight = [0.15 + ((i + 1) * GOLDEN % 1.0) ** 2 for i in range(n)]
    rest = total - n
    got = [1 + int(rest * w / sum(weight)) for w in weight]
    got[0] += total - sum(got)
    return got


def _spread(longest, n, empty=0):
    """n whole numbers up to `longest`, which the first one is; the last `empty` are 0."""
    got = [max(1, int(longest * (0.1 + 0.9 * (i * GOLDEN % 1.0)))) for i in range(n)]
    got[0] = longest
    return got[:n - empty] + [0] * empty


def _plan(case):
    """(tokens in the cache before, tokens this pass is about) of each sequence."""
    kind, b = case["kind"], case["batch"]
    if kind == "append":
        return [v - 1 for v in _spread(case["cached"], b)], _shares(case["tokens"], b)
    if kind == "read":
        return [0] * b, _shares(case["tokens"], b)
    if kind == "cache":
        return _spread(case["longest"], b, case["empty"]), [case["queries"]] * b
    return [case["prefix"] * (1 + i % 3) // 2 for i in range(b)], _shares(case["tokens"], b)


def _blocks(cached, new):
    """(first position of the first block that new tokens touch, positions up to the last new one)"""
    starts = [c // BLOCK * BLOCK for c in cached]
    return starts, [c + n - s for c, n, s in zip(cached, new, starts)]


def _sums(values):
    got = [0]
    for v in values:
        got.append(got[-1] + v)
    return got


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- inputs ----
def _heads(gen, tokens, heads, d, dtype, mean, spread):
    """Rows of heads with a direction that all tokens of a head share and a few loud dimensions."""
    x = torch.randn((tokens, heads, d), generator=gen, device="cuda").mul_(spread)
    x += mean * torch.randn((1, heads, d), generator=gen, device="cuda")
    x[:, :, torch.randint(0, d, (max(1, d // 64),), generator=gen, device="cuda")] *= 3
    return x.to(dtype)


def _whole(gen, shape, channel_mean):
    """Whole numbers of -127 .. 127: bells about a mean of their own for each head and dimension."""
    x = torch.empty(shape, dtype=torch.int8, device="cuda")
    mean = channel_mean * torch.randn((1, shape[1], 1, shape[3]), generator=gen, device="cuda")
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, shape[0], step):
        part = x[i:i + step]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(36).add_(mean).clamp_(-127, 127).round_())
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, b, d, kv = case["kind"], case["batch"], case["d"], case["kv"]
    dtype = DTYPES[case["dtype"]]
    before, now = _plan(case)
    s = dict(case=case, tokens=sum(now), cu=_ints(_sums(now)))
    if kind == "prompt":
        keys = [p + n for p, n in zip(before, now)]
        s["cu_k"], s["most_q"], s["most_k"] = _ints(_sums(keys)), max(now), max(keys)
        s["q"] = _heads(gen, sum(now), case["heads"], d, dtype, 0.5, 1.0)
        s["k"] = _heads(gen, sum(keys), kv, d, dtype, 0.5, 1.0)
        s["v"] = _heads(gen, sum(keys), kv, d, dtype, 0.5, 1.0)
        return s
    # the cache: pages in any order, tables longer than any sequence needs, -1 where no page is
    page = case["page"]
    held = [c + n for c, n in zip(before, now)] if kind != "cache" else before
    pages = [-(-h // page) for h in held]
    pool = sum(pages) + 1 + sum(pages) // 16
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((b, max(pages) + 2), -1, dtype=torch.int32, device="cuda")
    at = _sums(pages)
    for i in range(b):
        table[i, :pages[i]] = order[at[i]:at[i + 1]]
    s["table"], s["most"] = table, max(held)
    shape, scales = (pool, kv, page, d), (pool, kv, page // BLOCK)
    s["cache"] = (_whole(gen, shape, 8), _whole(gen, shape, 20),
                  torch.rand(scales, generator=gen, device="cuda").add_(0.5).mul_(1 / 36),
                  torch.rand(scales, generator=gen, device="cuda").add_(0.5).mul_(1 / 36))
    if kind == "cache":
        s["lengths"] = _ints(before)
        shape = (b, case["heads"], d) if case["queries"] == 1 else (b, case["queries"], case["heads"], d)
        s["q"] = _heads(gen, b * case["queries"], case["heads"], d, dtype, 0.5, 1.0).view(shape)
    elif kind == "read":
        s["starts"] = _ints(before)
    else:
        rot = case["rot"]
        # queries, keys and values as one projection leaves them, side by side
        s["qkv"] = _heads(gen, sum(now), case["heads"] + 2 * kv, d, dtype, 0.3, 1.0)
        angle = torch.arange(max(held), device="cuda").double()[:, None] * (
            10000.0 ** -(torch.arange(rot // 2, device="cuda").double() * 2 / rot))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["lengths"] = _ints(before)
        starts, counts = _blocks(before, now)
        s["starts"], s["touched"], s["cu_touched"] = _ints(starts), sum(counts), _ints(_sums(counts))
        s["most_new"], s["most_blocks"] = max(now), max(-(-c // BLOCK) for c in counts)
    return s


# ---- the plain forms ----
def _rows(cu, tokens):
    """(sequence, place in it) of each of the packed rows."""
    row = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), row, right=True)
    return seq, row - cu.long()[seq]


def _rotate(x, cos, sin, position, interleaved):
    rot = 2 * cos.shape[1]
    c, s = cos[position][:, None, :], sin[position][:, None, :]
    x = x.float()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _values(cache, scales, table, seq, position):
    """What the cache stands for at these positions: [rows, heads, d] in 32 bits."""
    page, at = cache.shape[2], position % cache.shape[2]
    number = table[seq, position // page].long()
    return cache[number, :, at].float() * scales[number, :, at // BLOCK][..., None]


def _store(x, cache, scales, s, seq, place):
    """New rows x [tokens, heads, d] in 32 bits into their blocks."""
    page, dims = cache.shape[2], x.shape[1:]
    b = s["table"].shape[0]
    wide = s["most_blocks"] * BLOCK
    # all positions of the blocks touched, and which of them are new
    offset = s["lengths"].long() - s["starts"].long()
    grid = torch.zeros((b, wide) + dims, device=x.device)
    fresh = torch.zeros((b, wide), dtype=torch.bool, device=x.device)
    grid[seq, offset[seq] + place] = x
    fresh[seq, offset[seq] + place] = True
    fresh = fresh.view(b, -1, BLOCK)
    grid = grid.view((b, -1, BLOCK) + dims)
    bi, ni = fresh.any(-1).nonzero(as_tuple=True)
    grid, fresh = grid[bi, ni], fresh[bi, ni]
    first = s["starts"].long()[bi] + ni * BLOCK
    number, at = s["table"][bi, first // page].long(), first % page
    # scales: of the new values, and of the block's older ones where it has some
    new = grid.abs().amax((1, 3)).clamp(min=TINY) / 127.0
    kept = ~fresh[:, 0]
    old = scales[number, :, at // BLOCK]
    scale = torch.where(kept[:, None], torch.maximum(new, old), new)
    ratio = torch.where(kept[:, None], old / scale, torch.ones_like(old))
    rows = at[:, None] + torch.arange(BLOCK, device=x.device)
    held = cache[number[:, None], :, rows].float()
    older = kept[:, None] & (torch.cumsum(fresh.int(), 1) == 0)
    values = torch.where(older[..., None, None], torch.round(held * ratio[:, None, :, None]), held)
    values = torch.where(fresh[..., None, None], torch.round(grid / scale[:, None, :, None]), values)
    cache[number[:, None], :, rows] = values.to(torch.int8)
    scales[number, :, at // BLOCK] = scale


def _plain_append(s):
    case = s["case"]
    heads, kv, dtype = case["heads"], case["kv"], s["qkv"].dtype
    q, k, v = s["qkv"].split((heads, kv, kv), 1)
    seq, place = _rows(s["cu"], s["tokens"])
    position = s["lengths"].long()[seq] + place
    q = _rotate(q, s["cos"], s["sin"], position, case["interleaved"])
    k = _rotate(k, s["cos"], s["sin"], position, case["interleaved"])
    kc, vc, ks, vs = s["cache"]
    _store(k, kc, ks, s, seq, place)
    _store(v.float(), vc, vs, s, seq, place)
    at, place = _rows(s["cu_touched"], s["touched"])
    position = s["starts"].long()[at] + place
    return (q.to(dtype), k.to(dtype), _values(kc, ks, s["table"], at, position).to(dtype),
            _values(vc, vs, s["table"], at, position).to(dtype))


def _plain_read(s):
    kc, vc, ks, vs = s["cache"]
    seq, place = _rows(s["cu"], s["tokens"])
    position, dtype = s["starts"].long()[seq] + place, DTYPES[s["case"]["dtype"]]
    return _values(kc, ks, s["table"], seq, position).to(dtype), _values(vc, vs, s["table"], seq, position).to(dtype)


def _attend(q, k, v, seen):
    """q [b, kv, rows, d], k and v [b, kv, keys, d], seen [b, 1, rows, keys]: 0 where nothing is seen."""
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(q.shape[-1]))
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_cache(s):
    case, n = s["case"], s["case"]["queries"]
    kc, vc, ks, vs = s["cache"]
    b, kv, d, most = case["batch"], case["kv"], case["d"], s["most"]
    group = case["heads"] // kv
    position = torch.arange(most, device="cuda").expand(b, most)
    seq = torch.arange(b, device="cuda")[:, None]
    number = s["table"][seq, position // case["page"]].long().clamp(min=0)
    at = position % case["page"]
    k = (kc[number, :, at].float() * ks[number, :, at // BLOCK][..., None]).transpose(1, 2)
    v = (vc[number, :, at].float() * vs[number, :, at // BLOCK][..., None]).transpose(1, 2)
    q = s["q"].float().view(b, n, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * group, d)
    last = s["lengths"].long()[:, None] - n + 1 + torch.arange(n, device="cuda").repeat_interleave(group)
    o = _attend(q, k, v, (position[:, None, :] < last[:, :, None])[:, None])
    return o.view(b, kv, n, group, d).permute(0, 2, 1, 3, 4).reshape(s["q"].shape).to(s["q"].dtype)


def _plain_prompt(s):
    case = s["case"]
    b, kv, d, heads = case["batch"], case["kv"], case["d"], case["heads"]
    mq, mk = s["most_q"], s["most_k"]
    seq, place = _rows(s["cu"], s["tokens"])
    kseq, kplace = _rows(s["cu_k"], s["k"].shape[0])
    q = torch.zeros((b, mq, heads, d), device="cuda")
    k, v = torch.zeros((2, b, mk, kv, d), device="cuda")
    q[seq, place], k[kseq, kplace], v[kseq, kplace] = s["q"].float(), s["k"].float(), s["v"].float()
    nq, nk = s["cu"].long().diff()[:, None, None], s["cu_k"].long().diff()[:, None, None]
    i, j = torch.arange(mq, device="cuda")[:, None], torch.arange(mk, device="cuda")
    seen = (i < nq) & (j < nk)
    if case["causal"]:
        seen = seen & (j - i <= nk - nq)
    group = heads // kv
    q = q.transpose(1, 2).reshape(b, kv, group * mq, d)
    o = _attend(q, k.transpose(1, 2), v.transpose(1, 2), seen[:, None].repeat(1, 1, group, 1))
    return o.view(b, heads, mq, d).transpose(1, 2)[seq, place].to(s["q"].dtype)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from megcc_b200 import ops
        if kind == "prompt":
            return ops.attention_prompt(state["q"], state["k"], state["v"], state["cu"], state["cu_k"],
                                        causal=case["causal"])
        cache = ops.KvCacheS8(*state["cache"])
        if kind == "cache":
            return ops.attention_cache_s8(state["q"], cache, state["table"], state["lengths"])
        if kind == "read":
            return ops.kv_read_s8(cache, state["table"], state["starts"], state["cu"], state["tokens"],
                                  DTYPES[case["dtype"]])
        q, k, v = state["qkv"].split((case["heads"], case["kv"], case["kv"]), 1)
        q, k = ops.kv_append_s8(cache, state["table"], state["lengths"], k, v, q, state["cos"], state["sin"],
                                cu_tokens=state["cu"], interleaved=case["interleaved"], turned_keys=True)
        # the blocks that changed, as the values they stand for
        return (q, k) + tuple(ops.kv_read_s8(cache, state["table"], state["starts"], state["cu_touched"],
                                             state["touched"], DTYPES[case["dtype"]]))
    return {"append": _plain_append, "read": _plain_read, "cache": _plain_cache, "prompt": _plain_prompt}[kind](state)


def work(case):
    before, now = _plan(case)
    kind, d, kv = case["kind"], case["d"], case["kv"]
    if kind == "append":
        n, heads = sum(now), case["heads"]
        counts = _blocks(before, now)[1]
        kept = sum(counts) - n
        return dict(bytes=2 * d * (n * (2 * heads + 3 * kv) + 2 * kv * sum(counts)) + 2 * kv * d * (n + kept) +
                    2 * n * case["rot"] * 2, flops=3.0 * n * (heads + kv) * case["rot"])
    if kind == "read":
        return dict(bytes=sum(now) * kv * (2 * d * 3 + 8 / BLOCK), flops=2.0 * sum(now) * kv * d)
    heads = case["heads"]
    if kind == "cache":
        n = case["queries"]
        pairs = sum(max(0, c - n + 1 + i) for c in before for i in range(n))
        return dict(bytes=sum(before) * kv * (2 * d + 8 / BLOCK) + 2 * 2 * case["batch"] * n * heads * d,
                    flops=4.0 * d * heads * pairs)
    keys = [p + n for p, n in zip(before, now)]
    pairs = sum(n * p + n * (n + 1) / 2 if case["causal"] else n * k for p, n, k in zip(before, now, keys))
    return dict(bytes=2 * d * (2 * heads * sum(now) + 2 * kv * sum(keys)), flops=4.0 * d * heads * pairs)


# ---- the same from the definitions, in 64 bits ----
def _exact_block(old, old_scale, new):
    """A block [tokens, d] of older whole numbers and new values: the values it stands for afterwards. Scales are
    numbers of 32 bits by definition."""
    top = new.abs().max(dim=0).values.max(dim=-1).values
    scale = (torch.where(top < TINY, torch.full_like(top, TINY), top) / 127).float()
    if len(old):
        scale = torch.where(old_scale > scale, old_scale, scale)
    wide = scale.double()[:, None]
    kept = (old.double() * (old_scale.double()[:, None] / wide)).round() if len(old) else old.double()
    return torch.cat((kept, (new / wide).round())) * wide


def _exact_append(s):
    case = s["case"]
    before, now = _plan(case)
    heads, kv, d, rot, page = case["heads"], case["kv"], case["d"], case["rot"], case["page"]
    q, k, v = s["qkv"].double().split((heads, kv, kv), 1)
    position = torch.cat([torch.arange(c, c + n) for c, n in zip(before, now)]).cuda()
    z = torch.complex(s["cos"].double()[position], s["sin"].double()[position])[:, None]

    def turn(x):
        y = x.clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (
            slice(0, rot // 2), slice(rot // 2, rot))
        w = torch.complex(x[..., first], x[..., second]) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y
    q, k = turn(q), turn(k)
    table = s["table"].cpu().tolist()
    got = []
    for new, whole, scales in ((k, s["cache"][0], s["cache"][2]), (v, s["cache"][1], s["cache"][3])):
        row, parts = 0, []
        for i, (c, n) in enumerate(zip(before, now)):
            p = c
            while p < c + n:
                first, end = p // BLOCK * BLOCK, min(c + n, p // BLOCK * BLOCK + BLOCK)
                number, at = table[i][first // page], first % page
                old = whole[number, :, at:at + p - first].transpose(0, 1)
                parts.append(_exact_block(old, scales[number, :, at // BLOCK], new[row:row + end - p]))
                row, p = row + end - p, end
        got.append(torch.cat(parts))
    return (q, k, got[0], got[1])


def _exact_keys(s, i, length, which):
    """Keys (0) or values (1) of sequence i: [length, heads, d]"""
    case = s["case"]
    pages = s["table"][i, :-(-length // case["page"])].long()
    x = s["cache"][which][pages].double()
    x = x.unflatten(2, (-1, BLOCK)) * s["cache"][which + 2][pages].double()[..., None, None]
    return x.flatten(2, 3).transpose(1, 2).reshape(-1, case["kv"], case["d"])[:length]


def _exact_attention(q, k, v, causal):
    """q [n, heads, d], k and v [m, kv, d] in 64 bits; the last query sees the last key."""
    n, m, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    o = torch.zeros_like(q)
    first = max(0, n - m) if causal else 0  # (rows in front see nothing)
    if m == 0 or n <= first:
        return o
    for h in range(q.shape[1]):
        a = q[first:, h] @ k[:, h // group].t() / math.sqrt(q.shape[2])
        if causal:
            hidden = torch.ones_like(a, dtype=torch.bool).triu(m - (n - first) + 1)
            a = a.masked_fill(hidden, -math.inf)
        o[first:, h] = torch.softmax(a, -1) @ v[:, h // group]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    before, now = _plan(case)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "read":
        return tuple(torch.cat([_exact_keys(s, i, n, w) for i, n in enumerate(now)]) for w in (0, 1))
    if case["kind"] == "cache":
        q = s["q"].double().view(case["batch"], case["queries"], case["heads"], case["d"])
        return torch.stack([_exact_attention(q[i], _exact_keys(s, i, n, 0), _exact_keys(s, i, n, 1), True)
                            for i, n in enumerate(before)]).view(s["q"].shape)
    keys = [p + n for p, n in zip(before, now)]
    return torch.cat([_exact_attention(q.double(), k.double(), v.double(), case["causal"]) for q, k, v in zip(
        s["q"].split(now), s["k"].split(keys), s["v"].split(keys))])
