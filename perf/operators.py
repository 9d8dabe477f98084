"""Performance cases of the int8 operators with scales found at run time: products with a scale per
token and per output channel, linear layers over float activations, mixture-of-experts layers for a
few tokens.

``listed()`` are fixed cases, ``draw()`` gives further ones of the same ranges; ``prepare`` makes what
a program holds before the call, ``run`` is one pass, ``work`` the bytes and operations the pass
cannot do without, ``exact`` its results in 64 bits. Where ``own`` is false ``run`` computes the plain
form from elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TINY = 2.0 ** -119   # the least magnitude a row's scale is taken from
GROUP = 32           # hidden units of an expert that share a scale


def _matmul(name, m, n, k, dtype, bias):
    return dict(name=name, kind="matmul", m=m, n=n, k=k, dtype=dtype, bias=bias)


def _linear(name, m, n, k, dtype, bias):
    return dict(name=name, kind="linear", m=m, n=n, k=k, dtype=dtype, bias=bias)


def _moe(name, t, d, f, e, top, dtype, renorm):
    return dict(name=name, kind="moe", t=t, d=d, f=f, e=e, top=top, dtype=dtype, renorm=renorm)


def listed():
    return [
        # One token of one sequence through a projection: its weights are read once, nothing else counts.
        _matmul("matmul_m1", 1, 4096, 4096, "bf16", False),
        # The classifier head of the model zoo over a small batch, logits in fp32.
        _matmul("matmul_classifier_m24", 24, 1000, 512, "f32", True),
        # A speculative or batched decoding step of an odd number of tokens through a wide projection.
        _matmul("matmul_m61", 61, 14336, 4096, "f16", False),
        # A short prompt, sizes that are no multiple of anything.
        _matmul("matmul_odd", 333, 4099, 2047, "f32", True),
        # A long prompt (or a training-sized batch of them): bound by the tensor cores.
        _matmul("matmul_m8192", 8192, 8192, 8192, "bf16", False),
        # One token, activations in 16 bits as the layer before leaves them.
        _linear("linear_m1", 1, 4096, 4096, "bf16", True),
        # A decoding step over a batch of sequences.
        _linear("linear_m128", 128, 4096, 11008, "bf16", False),
        # Prompts of several sequences, packed: a ragged number of rows.
        _linear("linear_m4001", 4001, 4096, 4096, "f16", True),
        # The smallest layer: one token, eight small experts.
        _moe("moe_t1_small", 1, 1024, 512, 8, 2, "f16", True),
        # One token through a wide layer of many experts.
        _moe("moe_t1", 1, 4096, 1536, 64, 8, "bf16", True),
        # A handful of tokens, sizes that fill no group and no tile.
        _moe("moe_t7_odd", 7, 1008, 344, 20, 3, "f16", False),
        # The largest few: nearly every expert has tokens.
        _moe("moe_t64", 64, 2048, 1024, 128, 8, "bf16", True),
    ]


def _log(rng, low, high, multiple=1):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, v // multiple * multiple)


def draw(rng):
    kind = rng.choice(["matmul", "linear", "moe"])
    dtype = rng.choice(["bf16", "f16"] if kind == "moe" else ["bf16", "f16", "f32"])
    while True:
        if kind == "moe":
            multiple = rng.choice([1, 8, 64, 64])
            t, e = _log(rng, 1, 64), _log(rng, 4, 128)
            d, f = _log(rng, 256, 4096, multiple), _log(rng, 128, 2048, multiple)
            top = rng.randint(1, min(8, e))
            if e * d * f <= 128 * 2048 * 1024 and t * top * d * f <= 64 * 8 * 2048 * 1024:
                return dict(kind=kind, t=t, d=d, f=f, e=e, top=top, dtype=dtype,
                            renorm=rng.random() < 0.5)
        else:
            multiple = rng.choice([1, 16, 128, 128])
            m = _log(rng, 1, 8192)
            n, k = _log(rng, 64, 16384, multiple), _log(rng, 64, 16384, multiple)
            if m * n * k <= 8192 ** 3 and m * n <= 8192 ** 2:
                return dict(kind=kind, m=m, n=n, k=k, dtype=dtype, bias=rng.random() < 0.5)


def _weights(gen, shape):
    """Quantised weights: their distribution is a bell over the whole range, clipped at its ends."""
    w = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat, step = w.view(-1), 1 << 26
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(40).clamp_(-127, 127).round_())
    return w


def _activations(gen, m, k, dtype):
    """Rows of unlike magnitude with a few channels that stand out, as residual streams have them."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((m, 1), generator=gen, device="cuda"))
    loud = torch.randint(0, k, (max(1, k // 512),), generator=gen, device="cuda")
    x[:, loud] *= 8
    return x.to(DTYPES[dtype])


def _scales(gen, shape, magnitude):
    return torch.rand(shape, generator=gen, device="cuda").add_(0.5).mul_(magnitude)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["kind"] == "moe":
        t, d, f, e = case["t"], case["d"], case["f"], case["e"]
        s["x"] = _activations(gen, t, d, case["dtype"])
        s["logits"] = torch.randn((t, e), generator=gen, device="cuda") * 1.5
        s["w1"], s["w2"] = _weights(gen, (e, 2 * f, d)), _weights(gen, (e, d, f))
        s["s1"] = _scales(gen, (e, 2 * f), 1 / (40 * math.sqrt(d)))
        s["s2"] = _scales(gen, (e, d), 1 / (40 * math.sqrt(f)))
    else:
        m, n, k = case["m"], case["n"], case["k"]
        if case["kind"] == "matmul":
            s["a"] = _weights(gen, (m, k))
            s["sa"] = _scales(gen, (m,), 1 / 40)
        else:
            s["x"] = _activations(gen, m, k, case["dtype"])
        s["b"] = _weights(gen, (n, k))
        s["sb"] = _scales(gen, (n,), 1 / (40 * math.sqrt(k)))
        s["bias"] = torch.randn((n,), generator=gen, device="cuda") if case["bias"] else None
    return s


# ---- the plain forms ----
def _quantize(x):
    """Values in -127 .. 127 and the factor they stand for, along the last axis: the product with the
    reciprocal is rounded once, to the nearest whole number (in 64 bits it is exact)."""
    amax = x.float().abs().amax(-1, keepdim=True).clamp(min=TINY)
    q = torch.round(x.double() * (127.0 / amax).double())
    return q, amax / 127.0


def _product(q, w):
    """Sums of products of whole numbers up to 127, exact: 64 bits hold them."""
    return torch.matmul(q.double(), w.double().transpose(-1, -2))


def _plain_matmul(a, sa, b, sb, bias, dtype):
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    if m * n * k <= 1 << 36:
        acc = _product(a, b).float()
    else:
        # whole numbers in 32 bits: sums over 1024 terms stay below 2^24 and are exact, their sums are not
        acc = torch.zeros((m, n), device=a.device)
        for i in range(0, k, 1024):
            acc += torch.matmul(a[:, i:i + 1024].float(), b[:, i:i + 1024].float().t())
    c = acc * sa[:, None] * sb[None, :]
    if bias is not None:
        c = c + bias
    return c.to(dtype)


def _route(logits, top, renorm):
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
    chosen = torch.gather(p, 1, order)
    return order, chosen / (chosen if renorm else p).sum(-1, keepdim=True)


def _plain_moe(s):
    case, x = s["case"], s["x"]
    f = case["f"]
    order, p = _route(s["logits"], case["top"], case["renorm"])
    xq, sx = _quantize(x)
    y = torch.zeros((case["t"], case["d"]), device=x.device)
    for j in range(case["top"]):
        e = order[:, j]
        z = _product(xq[:, None, :], s["w1"][e])[:, 0, :].float() * sx * s["s1"][e]
        g, u = z[:, :f], z[:, f:]
        h = g / (1 + torch.exp(-g)) * u
        pad = -f % GROUP
        h = torch.nn.functional.pad(h, (0, pad)).view(case["t"], -1, GROUP)
        hq, sh = _quantize(h)
        h = (hq * sh.double()).view(case["t"], -1)[:, :f]
        y += p[:, j:j + 1] * (_product(h[:, None, :], s["w2"][e])[:, 0, :].float() * s["s2"][e])
    return y.to(x.dtype)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from megcc_b200 import ops
        if kind == "matmul":
            return ops.matmul_s8_scaled(state["a"], state["b"], state["sa"], state["sb"],
                                        state["bias"], dtype=DTYPES[case["dtype"]])
        if kind == "linear":
            return ops.linear_s8(state["x"], state["b"], state["sb"], state["bias"])
        return ops.moe_s8(state["x"], state["logits"], state["w1"], state["s1"], state["w2"],
                          state["s2"], case["top"], renormalize=case["renorm"])
    if kind == "matmul":
        return _plain_matmul(state["a"], state["sa"], state["b"], state["sb"], state["bias"],
                             DTYPES[case["dtype"]])
    if kind == "linear":
        q, sx = _quantize(state["x"])
        return _plain_matmul(q, sx[:, 0], state["b"], state["sb"], state["bias"], state["x"].dtype)
    return _plain_moe(state)


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "moe":
        t, d, f, e, top = case["t"], case["d"], case["f"], case["e"], case["top"]
        # experts that at least one token chose, for tokens that choose alike by chance
        active = e * (1 - (1 - top / e) ** t)
        return dict(bytes=2 * t * d * size + 4 * t * e + active * (3 * d * f + 4 * (2 * f + d)),
                    flops=6.0 * t * top * d * f)
    m, n, k = case["m"], case["n"], case["k"]
    rows = m * k + 4 * m if case["kind"] == "matmul" else m * k * size
    return dict(bytes=rows + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * size,
                flops=2.0 * m * n * k)


# ---- the same from the definitions, in 64 bits ----
def _exact_rows(x):
    """(whole numbers, scale) of each row: scale and reciprocal are numbers of 32 bits by definition."""
    top = torch.maximum(x.max(-1).values, -x.min(-1).values)
    top = torch.where(top < TINY, torch.full_like(top, TINY), top)
    return (x * (127 / top).float().double()[..., None]).round(), (top / 127).float().double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "moe":
        if case["kind"] == "matmul":
            left = s["a"].double() * s["sa"].double()[:, None]
        else:
            q, scale = _exact_rows(s["x"].double())
            left = q * scale[:, None]
        c = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for i in range(0, case["n"], 2048):
            c[:, i:i + 2048] = left @ (s["b"][i:i + 2048].double() * s["sb"][i:i + 2048].double()[:, None]).t()
        return c if s["bias"] is None else c + s["bias"].double()
    f = case["f"]
    q, scale = _exact_rows(s["x"].double())
    x = q * scale[:, None]
    all_p = torch.softmax(s["logits"].double(), -1)
    y = torch.zeros((case["t"], case["d"]), dtype=torch.float64, device="cuda")
    for t, row in enumerate(s["logits"].cpu().tolist()):
        chosen = sorted(range(len(row)), key=lambda i: (-row[i], i))[:case["top"]]
        whole = all_p[t, chosen].sum() if case["renorm"] else 1.0
        for e in chosen:
            z = (s["w1"][e].double() * s["s1"][e].double()[:, None]) @ x[t]
            h = torch.sigmoid(z[:f]) * z[:f] * z[f:]
            for i in range(0, f, GROUP):
                q, scale = _exact_rows(h[i:i + GROUP])
                h[i:i + GROUP] = q * scale
            y[t] += all_p[t, e] / whole * ((s["w2"][e].double() * s["s2"][e].double()[:, None]) @ h)
    return y
