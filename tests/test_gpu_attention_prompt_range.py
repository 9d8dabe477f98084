"""Attention over whole prompts where its numbers lie far apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_attention_prompt import check, operands  # noqa: E402
from test_gpu_kv_cache import IDS, TYPES, sums  # noqa: E402


@pytest.mark.parametrize("up,scale", [(0, 0.0), (50, 0.0), (58, 0.0), (58, 2.0 ** -120), (59, -2.0 ** -121), (55, 2.0 ** -128),
                                      (20, 2.0 ** -43), (-40, 2.0 ** 78)])
def test_scales_of_large_and_small_scores(up, scale):
    """A scale of 0 makes all positions alike whatever the scores; the smallest ones are scales like any other."""
    for counts in ([200], [40, 129, 1]):
        q, k, v = operands(counts, counts, 4, 2, 64, torch.bfloat16)
        q, k = q * 2.0 ** up, k * 2.0 ** up
        assert bool(torch.isfinite(q).all() & torch.isfinite(k).all())
        check(ops.attention_prompt(q, k, v, sums(counts), scale=scale), q, k, v, counts, counts, True, scale)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,d", [(8, 1, 128), (16, 2, 64), (16, 1, 80), (32, 1, 64), (64, 1, 128), (64, 1, 48), (128, 1, 32),
                                        (24, 1, 64), (48, 3, 128)])
def test_groups_of_many_heads(heads, kv, d, causal, dtype):
    """Eight and more heads of a group share a tile: a few tokens each fill it."""
    for counts, keys in (([1, 3, 40, 0, 17], None), ([2, 70], [300, 129]), ([130], [5])):
        m = keys or counts
        q, k, v = operands(counts, m, heads, kv, d, dtype)
        got = ops.attention_prompt(q, k, v, sums(counts), None if keys is None else sums(keys), causal=causal)
        check(got, q, k, v, counts, m, causal)


def test_operands_of_more_than_two_to_the_31_elements():
    """A sequence at the far end of each; rows in front of it belong to none."""
    n, rows = 300, (1 << 23) + 300
    q, k, v = operands([n], [n], 2, 1, 128, torch.bfloat16)
    want = ops.attention_prompt(q, k, v, sums([n]))
    cu = torch.tensor([rows - n, rows], dtype=torch.int32, device="cuda")
    for in_front in (True, False):  # heads in front of tokens, or within
        big_q, big_out = (torch.empty((2, rows, 128) if in_front else (rows, 2, 128), dtype=torch.bfloat16, device="cuda")
                          for _ in range(2))
        if in_front:
            big_q, big_out = big_q.transpose(0, 1), big_out.transpose(0, 1)
        big_q[-n:] = q
        big_out[:-n] = 7
        cu_k = torch.tensor([2 * rows - n, 2 * rows], dtype=torch.int32, device="cuda")
        big_k, big_v = (torch.empty((2 * rows, 1, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        big_k[-n:], big_v[-n:] = k, v
        ops.attention_prompt(big_q, big_k, big_v, cu, cu_k, out=big_out)
        check(big_out[-n:], q, k, v, [n], [n], True)
        assert in_front or torch.equal(big_out[-n:], want)  # (heads in front are not packed: other tiles)
        assert bool((big_out[:-n] == 7).all())
        del big_q, big_out, big_k, big_v
