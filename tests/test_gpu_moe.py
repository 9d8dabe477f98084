"""The int8 mixture-of-experts layer against its definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_scaled import IDS, TYPES, gen, rows_of, whole  # noqa: E402

U = 2.0 ** -24


def layer(t, d, f, e, seed, dtype=torch.bfloat16):
    x = torch.randn((t, d), generator=gen(seed), device="cuda").to(dtype)
    logits = torch.randn((t, e), generator=gen(seed + 1), device="cuda") * 1.5
    w1, w2 = whole((e, 2 * f, d), seed + 2), whole((e, d, f), seed + 3)
    s1 = (torch.rand((e, 2 * f), generator=gen(seed + 4), device="cuda") + 0.5) / (74 * d ** 0.5)
    s2 = (torch.rand((e, d), generator=gen(seed + 5), device="cuda") + 0.5) / (74 * f ** 0.5)
    return x, logits, w1, s1, w2, s2


def definition(x, logits, w1, s1, w2, s2, top, renorm):
    """(y, how far an fp32 computation may be from it), 64 bits. Roundings, in steps of 2^-24 of the value:
    z three (its scale, its row's, the sum to fp32), h two more for the product and the quotient, 2 ulp = 4 for
    exp and one for its sum, and exp's argument moves by 3 |z|, all told 3 + 3 + 2 + 5 + 3 |z| <= 16 + 4 |z|; a
    group's maximum likewise. A number of h whose x * inv lies nearer to a half than that may come out one step
    away. A group's scale is 2 more off, a sum over g groups g + 8 warps, s_w2, p and their sum 4; p itself: the
    exponents' arguments |l| <= 32 give 64, exp 4, sums over 16 registers and 5 lanes 21, the quotient 1."""
    t, d = x.shape
    e, f = w2.shape[0], w2.shape[2]
    y = torch.zeros((t, d), dtype=torch.float64, device="cuda")
    off = torch.zeros_like(y)
    q, sx = rows_of(x)
    for i in range(t):
        row = logits[i].double()
        order = sorted(range(e), key=lambda j: (-float(row[j]), j))[:top]
        p = torch.softmax(row, 0)
        if renorm:
            p = p / p[order].sum()
        for j in order:
            if float(p[j]) == 0:
                continue
            z = (w1[j].double() @ q[i]) * sx[i].double() * s1[j].double()
            gate, up = z[:f], z[f:]
            h = gate / (1 + torch.exp(-gate)) * up
            pad = torch.nn.functional.pad(h, (0, -f % 32)).view(-1, 32)
            err = torch.nn.functional.pad((16 + 4 * gate.abs()) * U, (0, -f % 32)).view(-1, 32).amax(1, keepdim=True)
            amax = pad.abs().amax(1, keepdim=True).clamp(min=2.0 ** -119)
            r = pad * 127 / amax
            hq, sh = torch.round(r), amax / 127
            near = ((r.abs() % 1.0) - 0.5).abs() <= 127 * (2 * err + 4 * U)
            may = (near * sh).view(-1)[:f]
            part = (hq * sh).view(-1)[:f]
            rel = (err + 2 * U) * (hq.abs() * sh)
            may = may + rel.view(-1)[:f]
            w = w2[j].double() * s2[j].double()[:, None] * p[j]
            y[i] += w @ part
            sums = -(-f // 32) + 12 + 90 + top
            off[i] += w.abs() @ may + sums * U * (w.abs() @ part.abs())
    return y, off


def check(args, top, renorm, got=None):
    got = ops.moe_s8(*args, top, renorm) if got is None else got
    y, off = definition(*args, top, renorm)
    fi = torch.finfo(got.dtype)
    limit = off + (y.abs() + off) * (fi.eps / 2) + fi.tiny * fi.eps
    far = (got.double() - y).abs()
    assert bool((far <= limit).all()), float((far / limit).max())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("t,d,f,e,top", [(1, 64, 32, 1, 1), (1, 1024, 512, 8, 2), (2, 16, 8, 4, 4), (3, 100, 33, 5, 2),
                                         (7, 1008, 344, 20, 3), (8, 512, 96, 33, 8), (9, 130, 70, 3, 2),
                                         (17, 257, 129, 64, 16), (40, 320, 64, 2, 1), (64, 256, 128, 12, 5)])
def test_moe(t, d, f, e, top, renorm, dtype):
    check(layer(t, d, f, e, t + d, dtype), top, renorm)


def test_moe_of_wide_layers():
    check(layer(1, 4096, 1536, 16, 1), 8, True)
    check(layer(2, 16384, 64, 3, 2), 2, True)
    check(layer(10, 8192, 40, 3, 3), 1, False)
    check(layer(8, 16384, 40, 4, 6, torch.float32), 2, False)
    check(layer(5, 16383, 33, 3, 7), 3, True)
    check(layer(64, 8191, 32, 2, 8), 2, True)
    check(layer(4, 48, 5000, 3, 4), 2, True)
    check(layer(3, 64, 32, 512, 5), 16, True)


# every token at one expert; a token's experts alike with another's
def test_moe_of_tokens_that_choose_alike():
    x, logits, w1, s1, w2, s2 = layer(64, 192, 96, 6, 3)
    logits[:] = torch.tensor([0.0, 1.0, 5.0, -1.0, 3.0, 2.0], device="cuda")
    for top in (1, 3, 6):
        check((x, logits, w1, s1, w2, s2), top, True)


# ties go to the lowest index, -0 and 0 are equal, masked experts add nothing even where all are asked for
def test_moe_ties_and_masks():
    x, logits, w1, s1, w2, s2 = layer(5, 64, 64, 40, 4)
    logits[0] = 0
    logits[1] = 0
    logits[1, ::2] = -0.0
    logits[2] = float("-inf")
    logits[2, 7] = -3.0
    logits[3] = float("-inf")
    logits[4, 33:] = float("-inf")
    y = ops.moe_s8(x, logits, w1, s1, w2, s2, 4)
    assert bool((y[3] == 0).all())
    keep = [0, 1, 2, 4]
    for renorm in (True, False):
        y = ops.moe_s8(x, logits, w1, s1, w2, s2, 4, renorm)
        check((x[keep], logits[keep], w1, s1, w2, s2), 4, renorm, y[keep])
    # what is masked is not read into the result: experts whose scales are NaN
    s1[8:] = float("nan")
    s2[8:] = float("nan")
    y = ops.moe_s8(x, logits, w1, s1, w2, s2, 4)
    check((x[2:3], logits[2:3], w1, s1, w2, s2), 4, True, y[2:3])
    assert bool((y[3] == 0).all())


# The same behind the logits that a warp keeps in registers (128 of them)
@pytest.mark.parametrize("t", [1, 4, 12])
def test_moe_ties_and_masks_of_many_experts(t):
    x, logits, w1, s1, w2, s2 = layer(t, 48, 32, 300, 14)
    row = logits[t - 1]
    for renorm in (True, False):
        row[:] = 0                       # ties on both sides
        check((x, logits, w1, s1, w2, s2), 16, renorm)
        row[:] = -1
        row[130::7] = 2.5                # 25 ties, all behind
        row[200] = 3
        check((x, logits, w1, s1, w2, s2), 16, renorm)
        row[:] = float("-inf")
        row[290:] = torch.randn(10, generator=gen(15), device="cuda")
        check((x, logits, w1, s1, w2, s2), 16, renorm)
        row[:] = float("-inf")
        assert bool((ops.moe_s8(x, logits, w1, s1, w2, s2, 16, renorm)[t - 1] == 0).all())
        for bad in ("nan", "inf"):
            row[:] = 0
            row[299] = float(bad)
            y = ops.moe_s8(x, logits, w1, s1, w2, s2, 16, renorm)
            assert bool(y[t - 1].isnan().all()) and not bool(y[:t - 1].isnan().any())


# Two captured calls, replayed at once on two streams beside eager ones: each has a workspace of its own
def test_moe_graphs_at_once():
    args = [layer(t, 192, 96, 24, t) for t in (6, 40)]
    wants = [ops.moe_s8(*a, 4) for a in args]
    torch.cuda.synchronize()
    graphs = []
    for a in args:
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = [ops.moe_s8(*a, 4) for _ in range(5)]
        graphs.append((stream, graph, got))
    for _ in range(10):
        for stream, graph, got in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [ops.moe_s8(*a, 4) for a in args]
        torch.cuda.synchronize()
        for want, now, (_, _, got) in zip(wants, eager, graphs):
            assert torch.equal(now, want) and all(torch.equal(g, want) for g in got)


def test_moe_without_dependent_launches():
    from megcc_b200._lib import check as ok, lib
    args = [layer(t, 100, 40, 9, t) for t in (1, 7, 30)]
    wants = [ops.moe_s8(*a, 3) for a in args]
    ok(lib().mb200_set_option(b"pdl", 0))
    try:
        for a, want in zip(args, wants):
            assert torch.equal(ops.moe_s8(*a, 3), want)
    finally:
        ok(lib().mb200_set_option(b"pdl", 1))


@pytest.mark.parametrize("t", [4, 20])
def test_moe_of_special_values(t):
    x, logits, w1, s1, w2, s2 = layer(t, 96, 64, 8, 5, torch.float32)
    x[0, 95] = float("nan")
    x[1, 0] = float("inf")
    logits[2, 3] = float("nan")
    logits[t - 1, 0] = float("inf")
    y = ops.moe_s8(x, logits, w1, s1, w2, s2, 2)
    bad = [0, 1, 2, t - 1]
    assert bool(y[bad].isnan().all())
    rest = [i for i in range(t) if i not in bad]
    if rest:
        check((x[rest], logits[rest], w1, s1, w2, s2), 2, True, y[rest])
    x, logits, w1, s1, w2, s2 = layer(t, 96, 64, 8, 5)
    assert bool((ops.moe_s8(torch.zeros_like(x), logits, w1, s1, w2, s2, 2) == 0).all())
    assert ops.moe_s8(x[:0], logits[:0], w1, s1, w2, s2, 2).shape == (0, 96)


# Weights at any address, rows of x and y apart, the rows between them untouched, a workspace of any content
@pytest.mark.parametrize("offset,d,f", [(1, 96, 64), (8, 96, 72), (4, 112, 44), (0, 97, 31)])
def test_moe_operands_anywhere(offset, d, f):
    from megcc_b200._lib import MoeParam, check as ok, lib
    import ctypes
    t, e, top = 11, 6, 2
    x, logits, w1, s1, w2, s2 = layer(t, d, f, e, 6)
    b1 = torch.empty(w1.numel() + offset, dtype=torch.int8, device="cuda")[offset:].view_as(w1).copy_(w1)
    b2 = torch.empty(w2.numel() + offset, dtype=torch.int8, device="cuda")[offset:].view_as(w2).copy_(w2)
    wide = torch.zeros((t, d + offset + 5), device="cuda", dtype=x.dtype)
    wide[:, offset:offset + d] = x
    view = wide[:, offset:offset + d]
    check((x, logits, w1, s1, w2, s2), top, True, ops.moe_s8(view, logits, b1, s1, b2, s2, top))
    p = MoeParam(t, d, f, e, top, 1, 2)
    nbytes = lib().mb200_moe_s8_workspace_bytes(ctypes.byref(p))
    for fill in (0, 255):
        ws = torch.full((nbytes + 512,), fill, dtype=torch.uint8, device="cuda")
        base = ws.data_ptr() + -ws.data_ptr() % 256
        out = torch.full((t + 2, d + 3), 5.0, device="cuda", dtype=x.dtype)
        ok(lib().mb200_moe_s8(ctypes.byref(p), view.data_ptr(), view.stride(0), logits.data_ptr(), b1.data_ptr(),
                              s1.data_ptr(), b2.data_ptr(), s2.data_ptr(), out.data_ptr(), d + 3, base, nbytes,
                              ops._stream()))
        check((x, logits, w1, s1, w2, s2), top, True, out[:t, :d].clone())
        out[:t, :d] = 5.0
        assert bool((out == 5.0).all())
        assert bool((ws[base - ws.data_ptr() + nbytes:] == fill).all())


# The same bits every time, on another stream, captured and replayed with new tokens; a block of layers
# as it is used: linear, router, experts
@pytest.mark.parametrize("t", [1, 5, 33])
def test_block_with_router_streams_and_graphs(t):
    x, _, w1, s1, w2, s2 = layer(t, 256, 128, 16, 7)
    wl, sl = whole((256, 256), 8), torch.full((256,), 1e-3, device="cuda")
    router = torch.randn((256, 16), generator=gen(9), device="cuda")

    def block(x):
        h = ops.linear_s8(x, wl, sl)
        logits = ops.matmul_f32(h.float(), router)
        return h, logits, ops.moe_s8(h, logits, w1, s1, w2, s2, 4)

    h, logits, want = block(x)
    check((h, logits, w1, s1, w2, s2), 4, True, want)
    for _ in range(10):
        assert torch.equal(block(x)[2], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            replayed = block(x)
    for seed in (11, 12):
        x.copy_(torch.randn((t, 256), generator=gen(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed[2], block(x)[2])
