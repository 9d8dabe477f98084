"""The int8 mixture-of-experts layer at the corner where its first kernel's shared memory is fullest: deep rows at odd
places, more than eight tokens per expert, and many experts beside them."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from megcc_b200 import ops  # noqa: E402
from test_gpu_moe import check, layer  # noqa: E402


# (one expert fewer or more changes how many tokens a pass takes, and nothing else)
@pytest.mark.parametrize("t,e,top,d", [(64, 100, 16, 8191), (64, 127, 16, 8177), (64, 80, 16, 8191),
                                       (64, 81, 16, 8065), (63, 125, 16, 8191), (62, 123, 16, 8190),
                                       (64, 16, 16, 8191)])
def test_moe_of_deep_odd_rows_and_many_experts(t, e, top, d):
    check(layer(t, d, 33, e, e + t), top, True)


# the same for whole units of which none begins at a 16-byte address
def test_moe_of_deep_rows_at_odd_addresses():
    x, logits, w1, s1, w2, s2 = layer(64, 8192, 32, 100, 5)
    moved = torch.empty(w1.numel() + 1, dtype=torch.int8, device="cuda")[1:].view_as(w1).copy_(w1)
    check((x, logits, moved, s1, w2, s2), 16, False)
    check((x, logits, w1, s1, w2, s2), 16, False)


def test_moe_of_the_most_experts_and_deepest_rows():
    check(layer(64, 8191, 17, 512, 9), 16, True)
    check(layer(8, 16383, 17, 512, 10), 16, True)
    check(layer(4, 16383, 17, 512, 11, torch.float32), 16, True)
    x, logits, w1, s1, w2, s2 = layer(64, 8191, 32, 100, 12)
    want = ops.moe_s8(x, logits, w1, s1, w2, s2, 16)
    for _ in range(3):
        assert torch.equal(ops.moe_s8(x, logits, w1, s1, w2, s2, 16), want)
