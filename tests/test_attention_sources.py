"""What the attention kernels' sources must hold whatever the data, checked by reading them."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "megcc_b200", "csrc")


def test_warps_give_up_as_one():
    """A wait that runs out does so for a whole warp: lanes that went on alone would stop at the next instruction that wants all
    of them. Each bounded wait is voted on, or nothing depends on its outcome (those for what is still on its way at
    the end, which nobody may interrupt)."""
    with open(os.path.join(CSRC, "attention_prompt.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    waits = list(re.finditer(r"(.*)\bmbar_(?:try_)?wait\w*\(([^;]*);", text))
    assert len(waits) >= 4
    for w in waits:
        voted = "__all_sync(0xffffffffu, " in w.group(1)
        ignored = not w.group(1).strip() and w.group(2).rstrip(") ").endswith("&s_never")
        assert voted or ignored, w.group(0)
