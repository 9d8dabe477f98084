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
