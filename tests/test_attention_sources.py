"""What the attention kernels' sources must hold whatever the data, checked by reading them."""
import os
import re

import numpy as np
import pytest

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


def polynomials():
    """Coefficients of exp2_poly, highest first: (of fp16's, of bf16's)"""
    with open(os.path.join(CSRC, "attention_prompt.cu")) as f:
        body = re.search(r"float2 exp2_poly\(float2 x\) \{(.*?)\n\}", f.read(), re.S).group(1)
    fine, coarse = re.search(r"if constexpr \(fine\) \{(.*?)\} else \{(.*?)\}", body, re.S).groups()
    return [[np.float32(c) for c in re.findall(r"both\((-?[0-9.]+)f\)", part)] for part in (fine, coarse)]


@pytest.mark.parametrize("which,degree,bound", [(0, 4, 2.0 ** -18.5), (1, 3, 2.0 ** -13.7)])
def test_powers_by_polynomial(which, degree, bound):
    """2^f on [-1/2, 1/2] within the error that the results' bounds count with; Horner's steps round once each, 2^-24 of a number
    below 2^(1/2) (here: products and sums in 64 bits, then to 32, as an FMA does)."""
    coefficients = polynomials()[which]
    assert len(coefficients) == degree + 1
    f = np.linspace(-0.5, 0.5, 200001).astype(np.float32)
    p = np.full_like(f, coefficients[0])
    for c in coefficients[1:]:
        p = (p.astype(np.float64) * f.astype(np.float64) + np.float64(c)).astype(np.float32)
    exact = np.exp2(f.astype(np.float64))
    assert np.abs(p / exact - 1).max() <= bound + 2.0 ** -22
