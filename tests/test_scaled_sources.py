"""What the int8 operators with run-time scales hold in their sources."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "megcc_b200", "csrc")


# How many SMs there are is asked of the device: two levels of a choice of kernels that went by different counts would
# disagree about when a launch fills it.
@pytest.mark.parametrize("name", ["scaled_abi.cu", "scaled_stream.cu", "scaled_umma.cu", "moe_s8.cu", "stream_s8.cuh",
                                  "scaled_s8.cuh", "moe_s8.h"])
def test_the_number_of_sms_is_asked_for(name):
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"\b148\b", text)


# A launch that was refused is reported through refused(), which takes the runtime's record of it along.
@pytest.mark.parametrize("name", ["scaled_abi.cu", "scaled_stream.cu", "scaled_umma.cu", "moe_s8.cu"])
def test_refusals_of_the_runtime_take_its_error_along(name):
    with open(os.path.join(CSRC, name)) as f:
        assert "cudaGetErrorString" not in f.read()
